// The join of a block with its residual and the next block's norm (fhk_residual_norm) and its gradient.
//
//   y = x + s * gate * p, p = norm_post(f);  h = norm_pre(y);  norm(v) = n * w + b, n the normalised row
//
// Forward: one pass. LPR threads hold a row in registers (8 channels per chunk, NCH chunks per thread), so the mean,
// the variance (of the centred values, a second sum over registers) and the result need the row read once; x and f are
// read and y and h written once, which is the operator's floor. Long rows of many are bound by HBM (16384 x 4096, RMS norms:
// 90 us, 6.0 TB/s); short ones by instructions, 26 a value, and by the launch (130,000 x 64: 11 us, 6 TB/s; a layer norm with
// biases 13.5); a single row takes 4 us.
//
// Gradient: with d = dy + norm_pre'(dh) and q = s * gate * d,
//   norm'(dv) = r * (dn - n * mean(dn * n) [- mean(dn) for a layer norm]),  dn = dv * w
//   dx = d, df = norm_post'(q); dw_pre = sum dh * n_y, db_pre = sum dh.
// Every parameter gradient of the post side is formed from two column sums per gate row k, A1 = sum d * n_f and
// A0 = sum d: with Q = w A1 + b A0 (the column sum of d * p), dgate[k] = s Q[k], ds = sum_k gate[k] Q[k],
// dw_post = s sum_k gate[k] A1[k], db_post = s sum_k gate[k] A0[k]. So a thread keeps four sums per channel (two per
// side) for its columns over all rows of its CTA; a second kernel adds the CTAs' sums in a fixed order. The gradient is bound
// by instructions: 49 a value in 55 % of the issue slots, with 16 warps per SM because rows and sums fill the registers
// (16384 x 2048, RMS norms: 92 us with the sums, 4.4 TB/s; layer norms with biases 116).
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
// threads per SM that the registers are cut for: 128 each. Forward with 768 threads of 80 was 1 to 9 % faster at 513 to 1000
// channels and 5 to 10 % slower up to 200 and at 1024; with 1024 threads of 64 up to 40 % slower.
constexpr int kForwardThreads = 512, kGradThreads = 512;

// The sum over the LPR threads that share a row, in a fixed order, returned to all of them. LPR <= 32: within a warp;
// above: over the CTA (LPR == its threads), red holding one float per warp (every thread adds them up, by 16-byte reads).
template <int NW>
__device__ __forceinline__ float add_up(const float* red) {
    if (NW == 2) return red[0] + red[1];
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < NW; i += 4) {
        const float4 t = *reinterpret_cast<const float4*>(red + i);
        v += (t.x + t.y) + (t.z + t.w);
    }
    return v;
}
template <int LPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
    for (int o = (LPR < 32 ? LPR : 32) / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (LPR > 32) {
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
        __syncthreads();
        v = add_up<LPR / 32>(red);
    }
    return v;
}
// Two sums at once. The first exchange leaves each half of the lanes with one of them, so the rest of the tree is shared.
template <int LPR>
__device__ __forceinline__ float2 row_sum2(float a, float b, float* red) {
    constexpr int H = (LPR < 32 ? LPR : 32) / 2;
    const bool hi = threadIdx.x & H;
    float v = (hi ? b : a) + __shfl_xor_sync(0xffffffffu, hi ? a : b, H);
#pragma unroll
    for (int o = H / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (LPR > 32) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        if ((lane & 15) == 0) red[(lane ? 32 : 0) + warp] = v;
        __syncthreads();
        return make_float2(add_up<LPR / 32>(red), add_up<LPR / 32>(red + 32));
    }
    const float w = __shfl_xor_sync(0xffffffffu, v, H);
    return hi ? make_float2(w, v) : make_float2(v, w);
}

// x -> its normalised row n (in place; channels outside the row stay 0, all of them where the thread has no row);
// returns 1 / the deviation. red: 2 x 64 floats
template <int LPR, int NCH>
__device__ __forceinline__ void center(Chunk (&x)[NCH], const int (&valid)[NCH], float mean) {
#pragma unroll
    for (int k = 0; k < NCH; k++) {
#pragma unroll
        for (int j = 0; j < 4; j++) x[k].v[j] = __fadd2_rn(x[k].v[j], make_float2(-mean, -mean));
        x[k].cut(valid[k]);
    }
}
template <int NCH>
__device__ __forceinline__ float sum_of(const Chunk (&x)[NCH]) {
    float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < NCH; k++)
#pragma unroll
        for (int j = 0; j < 4; j++) s = __fadd2_rn(s, x[k].v[j]);
    return s.x + s.y;
}
template <int NCH>
__device__ __forceinline__ float squares_of(const Chunk (&x)[NCH]) {
    float2 q = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < NCH; k++)
#pragma unroll
        for (int j = 0; j < 4; j++) q = __ffma2_rn(x[k].v[j], x[k].v[j], q);
    return q.x + q.y;
}
template <int NCH>
__device__ __forceinline__ void scale_by(Chunk (&x)[NCH], const int (&valid)[NCH], float r) {
#pragma unroll
    for (int k = 0; k < NCH; k++) {
#pragma unroll
        for (int j = 0; j < 4; j++) x[k].v[j] = __fmul2_rn(x[k].v[j], make_float2(r, r));
        x[k].cut(valid[k]);  // r may be infinite
    }
}
template <int LPR, int NCH>
__device__ __forceinline__ float normalise(int kind, Chunk (&x)[NCH], const int (&valid)[NCH], float inv_c, float eps,
                                           float* red) {
    if (kind == FH_NORM_LAYER) center<LPR, NCH>(x, valid, row_sum<LPR>(sum_of(x), red) * inv_c);
    const float r = rsqrtf(row_sum<LPR>(squares_of(x), red + 64) * inv_c + eps);
    scale_by(x, valid, r);
    return r;
}
// two rows of the same thread at once, each sum of theirs together with the other's; a kind of none leaves its row as it is
template <int LPR, int NCH>
__device__ __forceinline__ float2 normalise2(int kx, Chunk (&x)[NCH], int ky, Chunk (&y)[NCH], const int (&valid)[NCH],
                                             float inv_c, float eps, float* red) {
    if (kx == FH_NORM_LAYER || ky == FH_NORM_LAYER) {
        const float2 s = row_sum2<LPR>(sum_of(x), sum_of(y), red);
        if (kx == FH_NORM_LAYER) center<LPR, NCH>(x, valid, s.x * inv_c);
        if (ky == FH_NORM_LAYER) center<LPR, NCH>(y, valid, s.y * inv_c);
    }
    const float2 q = row_sum2<LPR>(squares_of(x), squares_of(y), red + 64);
    const float2 r = make_float2(rsqrtf(q.x * inv_c + eps), rsqrtf(q.y * inv_c + eps));
    if (kx != FH_NORM_NONE) scale_by(x, valid, r.x);
    if (ky != FH_NORM_NONE) scale_by(y, valid, r.y);
    return r;
}

// How rows fill the threads that hold them: every chunk whole in every thread (no masks), chunks whole or absent, or a last
// one partly filled. The masks are a third of the instructions where they are not needed.
constexpr int kAny = 0, kWholeChunks = 1, kFull = 2;
template <int FILL>
__device__ __forceinline__ int channels_of(int left) {
    return FILL == kFull ? 8 : FILL == kWholeChunks ? (left > 0 ? 8 : 0) : max(0, min(8, left));
}

// by (plus) a vector's channels `at`; none: unchanged
template <typename T>
__device__ __forceinline__ void mul_vec(Chunk& x, const void* w, long long at, int valid, bool vec = true) {
    if (!w) return;
    const Chunk t = load_chunk(static_cast<const T*>(w) + at, valid, vec);
#pragma unroll
    for (int j = 0; j < 4; j++) x.v[j] = __fmul2_rn(x.v[j], t.v[j]);
}
template <typename T>
__device__ __forceinline__ void add_vec(Chunk& x, const void* w, long long at, int valid) {
    if (!w) return;
    const Chunk t = load_chunk(static_cast<const T*>(w) + at, valid);
#pragma unroll
    for (int j = 0; j < 4; j++) x.v[j] = __fadd2_rn(x.v[j], t.v[j]);
}
__device__ __forceinline__ void add(Chunk& x, const Chunk& y) {
#pragma unroll
    for (int j = 0; j < 4; j++) x.v[j] = __fadd2_rn(x.v[j], y.v[j]);
}
__device__ __forceinline__ void mul(Chunk& x, const Chunk& y) {
#pragma unroll
    for (int j = 0; j < 4; j++) x.v[j] = __fmul2_rn(x.v[j], y.v[j]);
}
__device__ __forceinline__ void add_product(Chunk& x, const Chunk& a, const Chunk& b) {
#pragma unroll
    for (int j = 0; j < 4; j++) x.v[j] = __ffma2_rn(a.v[j], b.v[j], x.v[j]);
}
// whether every gate row begins on a 16-byte boundary
template <typename P>
__device__ __forceinline__ bool gate_vec(const P& p) {
    return (p.gate_pitch & 7) == 0 && ((uintptr_t)p.gate & 15) == 0;
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
    __device__ __forceinline__ void copy(int stage, int tensor, int k, const T* src, int valid) const {
        const uint32_t dst = (uint32_t)__cvta_generic_to_shared(slot(stage, tensor, k));
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(2 * valid) : "memory");
    }
    static __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
    static __device__ __forceinline__ void wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(STAGES - 2) : "memory"); }
    __device__ __forceinline__ Chunk read(int stage, int tensor, int k) const { return unpack<T>(*slot(stage, tensor, k)); }
};

// Chunks that a thread keeps for itself in shared memory, as 32-bit values
template <int THREADS>
struct Kept {
    float4* buf;
    static constexpr size_t kChunkBytes = (size_t)THREADS * 32;  // one chunk of every thread
    __device__ __forceinline__ Chunk get(int i) const {
        const float4 a = buf[2 * i * THREADS + threadIdx.x], b = buf[(2 * i + 1) * THREADS + threadIdx.x];
        Chunk x;
        x.v[0] = make_float2(a.x, a.y), x.v[1] = make_float2(a.z, a.w);
        x.v[2] = make_float2(b.x, b.y), x.v[3] = make_float2(b.z, b.w);
        return x;
    }
    __device__ __forceinline__ void put(int i, const Chunk& x) const {
        buf[2 * i * THREADS + threadIdx.x] = make_float4(x.v[0].x, x.v[0].y, x.v[1].x, x.v[1].y);
        buf[(2 * i + 1) * THREADS + threadIdx.x] = make_float4(x.v[2].x, x.v[2].y, x.v[3].x, x.v[3].y);
    }
};

// THREADS / LPR rows at a time per CTA
template <typename T, int THREADS, int LPR, int NCH, int STAGES, int FILL>
__global__ void __launch_bounds__(THREADS, kForwardThreads / THREADS) k_residual_norm(const FhResidualNormParams p, unsigned rows_per_gate) {
    __shared__ __align__(16) float red[2 * 4 * 64];
    extern __shared__ uint4 ring_mem[];
    const Ring<T, THREADS, NCH, 2, STAGES> ring{ring_mem};
    constexpr int RPC = THREADS / LPR;
    const int l = threadIdx.x % LPR, sub = threadIdx.x / LPR;
    const float inv_c = 1.0f / (float)p.c;
    int valid[NCH];
#pragma unroll
    for (int k = 0; k < NCH; k++) valid[k] = channels_of<FILL>(p.c - 8 * (l + k * LPR));
    const bool gvec = gate_vec(p), has_f = p.f != nullptr, has_h = p.h != nullptr;
    const int first = blockIdx.x * RPC + sub, step = gridDim.x * RPC, m = (int)p.m;
    // running pointers: the row that is copied, and the row that is written
    const T* x = static_cast<const T*>(p.x) + first * p.x_pitch + 8 * l;
    const T* f = static_cast<const T*>(p.f) + first * p.f_pitch + 8 * l;
    T* y = static_cast<T*>(p.y) + first * p.y_pitch + 8 * l;
    T* h = static_cast<T*>(p.h) + first * p.h_pitch + 8 * l;
    long long ahead = first;
    auto fetch = [&](int stage) {
        const bool on = ahead < m;
#pragma unroll
        for (int k = 0; k < NCH; k++) {
            const int vk = on ? valid[k] : 0;
            ring.copy(stage, 0, k, vk ? x + 8 * k * LPR : static_cast<const T*>(p.x), vk);
            if (has_f) ring.copy(stage, 1, k, vk ? f + 8 * k * LPR : static_cast<const T*>(p.f), vk);
        }
        ring.commit();
        ahead += step;
        x += step * p.x_pitch;
        f += step * p.f_pitch;
    };
#pragma unroll
    for (int q = 0; q < STAGES - 1; q++) fetch(q);
    // a channel's factors, kept from row to row: w_post * scale * gate and b_post * scale * gate (while the gate's row stays
    // the same), w_pre and (where a thread has one chunk) b_pre
    constexpr bool HOIST = NCH == 1;
    Chunk post_w[NCH], post_b[NCH], pre_w[NCH], pre_b[HOIST ? NCH : 1];
    auto fold = [&](const T* gate) {
#pragma unroll
        for (int k = 0; k < NCH; k++) {
            const int c = 8 * (l + k * LPR);
            Chunk s;
#pragma unroll
            for (int j = 0; j < 4; j++) s.v[j] = make_float2(1.0f, 1.0f);
            post_b[k].zero();
            if (valid[k]) {
                mul_vec<T>(s, p.scale, c, valid[k]);
                mul_vec<T>(s, gate, c, valid[k], gvec);
                add_vec<T>(post_b[k], p.b_post, c, valid[k]);
                mul(post_b[k], s);
                mul_vec<T>(s, p.w_post, c, valid[k]);
            }
            post_w[k] = s;
        }
    };
#pragma unroll
    for (int k = 0; k < NCH; k++) {
#pragma unroll
        for (int j = 0; j < 4; j++) pre_w[k].v[j] = make_float2(1.0f, 1.0f);
        if (HOIST) pre_b[HOIST ? k : 0].zero();
        if (!valid[k]) continue;
        mul_vec<T>(pre_w[k], p.w_pre, 8 * (l + k * LPR), valid[k]);
        if (HOIST) add_vec<T>(pre_b[HOIST ? k : 0], p.b_pre, 8 * (l + k * LPR), valid[k]);
    }
    int gate_row = -1;
    if (has_f && !p.gate) fold(nullptr);
    int stage = 0;
    // every thread of a CTA runs the same number of iterations: the sums are CTA-wide barriers or whole-warp shuffles.
    // A row's sums use the buffers of its parity: between a buffer's uses lies a barrier of the row between them.
    float* sums = red;
    for (long long row = first; row - sub < m; row += step) {
        Chunk xv[NCH], fv[NCH];
        int vr[NCH];  // the channels of this thread's row
        ring.wait();
#pragma unroll
        for (int k = 0; k < NCH; k++) {
            vr[k] = (FILL == kFull && RPC == 1) || row < m ? valid[k] : 0;
            xv[k] = ring.read(stage, 0, k);
            if (has_f) fv[k] = ring.read(stage, 1, k);
        }
        fetch(stage == 0 ? STAGES - 1 : stage - 1);
        stage = stage + 1 == STAGES ? 0 : stage + 1;
        if (has_f) {
            if (p.post != FH_NORM_NONE) normalise<LPR, NCH>(p.post, fv, vr, inv_c, p.eps, sums);
            const T* gate = static_cast<const T*>(p.gate);
            if (gate) {
                const int at = (unsigned)min((int)row, m - 1) / rows_per_gate;
                gate += at * p.gate_pitch;
                if (at != gate_row) fold(gate), gate_row = at;
            }
#pragma unroll
            for (int k = 0; k < NCH; k++) {
                if (!vr[k]) continue;
                add_product(xv[k], fv[k], post_w[k]);
                if (p.b_post) add(xv[k], post_b[k]);
                store_chunk(y + 8 * k * LPR, vr[k], xv[k]);
            }
            y += step * p.y_pitch;
        }
        if (has_h) {
            normalise<LPR, NCH>(p.pre, xv, vr, inv_c, p.eps, sums + 128);
#pragma unroll
            for (int k = 0; k < NCH; k++) {
                if (!vr[k]) continue;
                mul(xv[k], pre_w[k]);
                if constexpr (HOIST) add(xv[k], pre_b[k]);
                else add_vec<T>(xv[k], p.b_pre, 8 * (l + k * LPR), vr[k]);
                store_chunk(h + 8 * k * LPR, vr[k], xv[k]);
            }
            h += step * p.h_pitch;
        }
        sums = sums == red ? red + 256 : red;
    }
}

// dn -> the gradient of the row that n was normalised from
template <int LPR, int NCH>
__device__ __forceinline__ void normalise_grad(int kind, Chunk (&dn)[NCH], const Chunk (&n)[NCH], float r, float inv_c, float* red) {
    float2 s1 = make_float2(0.0f, 0.0f), s0 = s1;
#pragma unroll
    for (int k = 0; k < NCH; k++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            s1 = __ffma2_rn(dn[k].v[j], n[k].v[j], s1);
            s0 = __fadd2_rn(s0, dn[k].v[j]);
        }
    const float2 s = row_sum2<LPR>(s1.x + s1.y, s0.x + s0.y, red);
    const float m1 = -s.x * inv_c, m0 = kind == FH_NORM_LAYER ? -s.y * inv_c : 0.0f;
#pragma unroll
    for (int k = 0; k < NCH; k++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float2 t = __ffma2_rn(n[k].v[j], make_float2(m1, m1), __fadd2_rn(dn[k].v[j], make_float2(m0, m0)));
            dn[k].v[j] = __fmul2_rn(t, make_float2(r, r));
        }
}

// How a gradient's rows are shared out. Gate rows are `groups` runs of `len` rows. With few of them each run is cut
// into `slices` and a CTA takes one slice; with many a CTA takes `per_cta` whole runs one after another and finishes
// their dgate rows itself (slices == 1).
struct Split {
    long long len;
    int groups, slices, per_cta, ctas;
    bool whole;   // CTAs finish their runs' dgate
    bool zeroth;  // sum d and sum dh are wanted (a bias is there, or its gradient)
};

// the CTA's column sums, part [cta][4][c]: (A1, A0), or with whole runs (sum gate A1, sum gate A0); then sum dh n_y, sum dh
template <typename T, int THREADS, int LPR, int NCH, int STAGES, bool WHOLE, int FILL, bool ZEROTH>
__global__ void __launch_bounds__(THREADS, kGradThreads / THREADS) k_residual_norm_grad(const FhResidualNormGradParams p, const Split sp,
                                                                 float* part) {
    constexpr int RPC = THREADS / LPR;
    __shared__ __align__(16) float red[2 * 6 * 64];  // whole 128-byte lines: the ring behind it is read by whole lines (2 % of the time)
    float* sums = red;  // a row's sums use the buffers of its parity, as in the forward kernel
    __shared__ float fold[RPC > 1 ? THREADS * NCH * 8 : 1];
    extern __shared__ uint4 ring_mem[];
    const Ring<T, THREADS, NCH, 4, STAGES> ring{ring_mem};
    // With two chunks a thread, what its registers cannot hold beside the rows: a channel's post factor at [k], sum d and
    // sum dh at [NCH + k] and [2 NCH + k]. In registers more of the row's values spilled: 4096 x 8192 with biases 257 us, 230
    // so. 64 to 144 bytes a thread still do (404 with whole runs, where those of one chunk spill 16 to 32)
    constexpr bool SHARED = NCH > 1;
    const Kept<THREADS> kept{reinterpret_cast<float4*>(ring_mem + Ring<T, THREADS, NCH, 4, STAGES>::kBytes / 16)};
    const int l = threadIdx.x % LPR, sub = threadIdx.x / LPR;
    const float inv_c = 1.0f / (float)p.c;
    int valid[NCH];
#pragma unroll
    for (int k = 0; k < NCH; k++) valid[k] = channels_of<FILL>(p.c - 8 * (l + k * LPR));
    const T* f = static_cast<const T*>(p.f);
    const bool gvec = gate_vec(p);
    pdl_trigger();  // what follows sums this kernel's parts, once all of it has ended
    constexpr int Z = ZEROTH && !SHARED ? NCH : 1;
    Chunk a1[NCH], a0[Z], b1[NCH], b0[Z], g1[WHOLE ? NCH : 1], g0[WHOLE ? NCH : 1];
    auto set = [&](Chunk (&sum)[Z], int at, int k, const Chunk& x) {
        if constexpr (SHARED) kept.put(at + k, x);
        else sum[k] = x;
    };
    auto add_to = [&](Chunk (&sum)[Z], int at, int k, const Chunk& x) {
        if constexpr (SHARED) {
            Chunk t = kept.get(at + k);
            add(t, x);
            kept.put(at + k, t);
        } else {
            add(sum[k], x);
        }
    };
    auto get = [&](const Chunk (&sum)[Z], int at, int k) {
        if constexpr (SHARED) return kept.get(at + k);
        else return sum[k];
    };
    constexpr int kA0 = NCH, kB0 = 2 * NCH;  // where sum d and sum dh are kept
#pragma unroll
    for (int k = 0; k < NCH; k++) {
        a1[k].zero(), b1[k].zero();
        if (ZEROTH) set(a0, kA0, k, a1[k]), set(b0, kB0, k, b1[k]);
        if (WHOLE) g1[k].zero(), g0[k].zero();
    }
    // v summed over the CTA's row groups (in order), returned to all of them
    auto over_rows = [&](Chunk& x) {
        if (RPC == 1) return;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; j++) fold[(sub * 8 + j) * LPR + l] = x.get(j);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; j++) {
            float s = 0.0f;
#pragma unroll 4
            for (int i = 0; i < RPC; i++) s += fold[(i * 8 + j) * LPR + l];
            x.set(j, s);
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
        const T* tp[4] = {static_cast<const T*>(p.dy), static_cast<const T*>(p.dh), static_cast<const T*>(p.y), f};
        const long long pitch[4] = {p.dy_pitch, p.dh_pitch, p.y_pitch, p.f_pitch};
        const bool has[4] = {p.dy != nullptr, p.dh != nullptr, p.dh != nullptr, f != nullptr};
        const T* const tp0[4] = {tp[0], tp[1], tp[2], tp[3]};
#pragma unroll
        for (int t = 0; t < 4; t++) tp[t] += (lo + sub) * pitch[t] + 8 * l;
        T* dx = static_cast<T*>(p.dx) + (lo + sub) * p.dx_pitch + 8 * l;
        T* df = static_cast<T*>(p.df) + (lo + sub) * p.df_pitch + 8 * l;
        long long ahead = lo + sub;
        auto fetch = [&](int stage) {
            const bool on = ahead < hi;
#pragma unroll
            for (int t = 0; t < 4; t++) {
                if (!has[t]) continue;
#pragma unroll
                for (int k = 0; k < NCH; k++) {
                    const int vk = on ? valid[k] : 0;
                    ring.copy(stage, t, k, vk ? tp[t] + 8 * k * LPR : tp0[t], vk);
                }
                tp[t] += RPC * pitch[t];
            }
            ring.commit();
            ahead += RPC;
        };
        if (WHOLE) asm volatile("cp.async.wait_all;\n" ::: "memory");  // the last run's copies, before their slots are reused
#pragma unroll
        for (int q = 0; q < STAGES - 1; q++) fetch(q);
        int stage = 0;
        // what a channel's values are multiplied by in every row of the run: scale * gate * w_post, and w_pre (which two
        // chunks a thread read again for each row)
        Chunk post_w[NCH], pre_w[NCH];
#pragma unroll
        for (int k = 0; k < NCH; k++) {
            const int c = 8 * (l + k * LPR);
#pragma unroll
            for (int j = 0; j < 4; j++) post_w[k].v[j] = pre_w[k].v[j] = make_float2(1.0f, 1.0f);
            if (valid[k]) {
                mul_vec<T>(post_w[k], p.scale, c, valid[k]);
                if (p.gate) mul_vec<T>(post_w[k], p.gate, (long long)grp * p.gate_pitch + c, valid[k], gvec);
                mul_vec<T>(post_w[k], p.w_post, c, valid[k]);
                if (!SHARED) mul_vec<T>(pre_w[k], p.w_pre, c, valid[k]);
            }
            if (SHARED) kept.put(k, post_w[k]);
        }
        for (long long row = lo + sub; row - sub < hi; row += RPC) {
            Chunk d[NCH], dh[NCH], yv[NCH], fv[NCH];
            int vr[NCH];  // the channels of this thread's row
            ring.wait();
#pragma unroll
            for (int k = 0; k < NCH; k++) {
                vr[k] = (FILL == kFull && RPC == 1) || row < hi ? valid[k] : 0;
                if (has[0]) d[k] = ring.read(stage, 0, k);
                else d[k].zero();
                if (has[1]) {
                    dh[k] = ring.read(stage, 1, k);
                    yv[k] = ring.read(stage, 2, k);
                } else {
                    yv[k].zero();
                }
                if (has[3]) fv[k] = ring.read(stage, 3, k);
                else fv[k].zero();
            }
            fetch(stage == 0 ? STAGES - 1 : stage - 1);
            stage = stage + 1 == STAGES ? 0 : stage + 1;
            const int kind_y = has[1] ? p.pre : FH_NORM_NONE;
            float2 r = make_float2(1.0f, 1.0f);
            if (kind_y != FH_NORM_NONE || p.post != FH_NORM_NONE)
                r = normalise2<LPR, NCH>(kind_y, yv, p.post, fv, vr, inv_c, p.eps, sums);
            if (has[1]) {
#pragma unroll
                for (int k = 0; k < NCH; k++) {
                    add_product(b1[k], dh[k], yv[k]);
                    if (ZEROTH) add_to(b0, kB0, k, dh[k]);
                    if constexpr (!SHARED) mul(dh[k], pre_w[k]);
                    else if (vr[k]) mul_vec<T>(dh[k], p.w_pre, 8 * (l + k * LPR), vr[k]);
                }
                normalise_grad<LPR, NCH>(p.pre, dh, yv, r.x, inv_c, sums + 128);
#pragma unroll
                for (int k = 0; k < NCH; k++)
                    if (vr[k]) {
                        add(d[k], dh[k]);
                        d[k].cut(vr[k]);
                    }
            }
            if (p.dx) {
#pragma unroll
                for (int k = 0; k < NCH; k++)
                    if (vr[k]) store_chunk(dx + 8 * k * LPR, vr[k], d[k]);
                dx += RPC * p.dx_pitch;
            }
            if (has[3]) {
#pragma unroll
                for (int k = 0; k < NCH; k++) {
                    add_product(a1[k], d[k], fv[k]);
                    if (ZEROTH) add_to(a0, kA0, k, d[k]);
                    if constexpr (SHARED) mul(d[k], kept.get(k));
                    else mul(d[k], post_w[k]);
                }
                if (p.df) {
                    if (p.post != FH_NORM_NONE) normalise_grad<LPR, NCH>(p.post, d, fv, r.y, inv_c, sums + 256);
#pragma unroll
                    for (int k = 0; k < NCH; k++)
                        if (vr[k]) store_chunk(df + 8 * k * LPR, vr[k], d[k]);
                    df += RPC * p.df_pitch;
                }
            }
            sums = sums == red ? red + 384 : red;
        }
        if (WHOLE) {  // the run's dgate row, and its share of the sums over gate rows
            const long long grow = p.gate ? (long long)grp * p.gate_pitch : 0;
#pragma unroll
            for (int k = 0; k < (WHOLE ? NCH : 1); k++) {
                const int c = 8 * (l + k * LPR);
                Chunk zeroth = get(a0, kA0, k);
                over_rows(a1[k]);
                over_rows(zeroth);
                if (valid[k] && sub == 0) {
                    if (p.dgate) {
                        Chunk q = a1[k], w0 = zeroth;
                        mul_vec<T>(q, p.w_post, c, valid[k]);
                        if (p.b_post) {
                            mul_vec<T>(w0, p.b_post, c, valid[k]);
                            add(q, w0);
                        }
                        mul_vec<T>(q, p.scale, c, valid[k]);
                        store_chunk(static_cast<T*>(p.dgate) + (long long)grp * p.dgate_pitch + c, valid[k], q,
                                    (p.dgate_pitch & 7) == 0 && ((uintptr_t)p.dgate & 15) == 0);
                    }
                    mul_vec<T>(a1[k], p.gate, grow + c, valid[k], gvec);
                    mul_vec<T>(zeroth, p.gate, grow + c, valid[k], gvec);
                }
                if (sub == 0) {  // every row group of the CTA holds the run's whole sum: the first keeps it
                    add(g1[k], a1[k]);
                    add(g0[k], zeroth);
                }
                a1[k].zero();
                set(a0, kA0, k, a1[k]);
            }
        }
    }
    asm volatile("cp.async.wait_all;\n" ::: "memory");

    // the CTA's sums
    float* out = part + (long long)blockIdx.x * 4 * p.c;
    auto put = [&](int q, auto value, bool summed) {
#pragma unroll
        for (int k = 0; k < NCH; k++) {
            Chunk x = value(k);
            if (!summed) over_rows(x);
            const int c = 8 * (l + k * LPR);
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (sub == 0 && j < valid[k]) out[(long long)q * p.c + c + j] = x.get(j);
        }
    };
    if constexpr (WHOLE) {
        put(0, [&](int k) { return g1[k]; }, true);
        put(1, [&](int k) { return g0[k]; }, true);
    } else {
        put(0, [&](int k) { return a1[k]; }, false);
        if constexpr (ZEROTH) put(1, [&](int k) { return get(a0, kA0, k); }, false);
    }
    put(2, [&](int k) { return b1[k]; }, false);
    if constexpr (ZEROTH) put(3, [&](int k) { return get(b0, kB0, k); }, false);
}

// 16 columns per CTA, 64 threads per column over the CTAs' sums; blockIdx.y: 0 the post side, 1 the pre side. Up to 64 gate
// rows at a time, each one's CTAs shared out over 64 / rows threads, whose sums are added in order.
template <typename T>
__global__ void __launch_bounds__(1024) k_residual_norm_params(const FhResidualNormGradParams p, const Split sp,
                                                               const float* part) {
    __shared__ float2 s[64][17];
    const int lane = threadIdx.x & 15, w = threadIdx.x >> 4, col = blockIdx.x * 16 + lane;
    const bool on = col < p.c, post = blockIdx.y == 0;
    auto at = [&](const void* v, long long i, float none) { return v && on ? Elem<T>::to(static_cast<const T*>(v)[i]) : none; };
    auto put = [&](void* v, long long i, float x) {
        if (v && on) static_cast<T*>(v)[i] = Elem<T>::from(x);
    };
    // the pre side and whole runs are one sum over all CTAs
    const int groups = post && !sp.whole ? sp.groups : 1, slices = sp.ctas / groups;
    const float wp = at(p.w_post, col, 1.0f), bp = at(p.b_post, col, 0.0f), sc = at(p.scale, col, 1.0f);
    pdl_wait();
    float g1 = 0.0f, g0 = 0.0f;
    for (int k0 = 0; k0 < groups; k0 += 64) {
        const int batch = min(64, groups - k0), parts = 64 / batch;
        float2 v = make_float2(0.0f, 0.0f);
        if (on && w < batch * parts) {
            const int k = k0 + w / parts, q = w % parts;
            const float* src = part + (post ? 0 : 2 * (long long)p.c) + col;
            const int lo = k * slices + slices * q / parts, hi = k * slices + slices * (q + 1) / parts;
#pragma unroll 8
            for (int i = lo; i < hi; i++) {
                v.x += src[(long long)i * 4 * p.c];
                if (sp.zeroth) v.y += src[(long long)i * 4 * p.c + p.c];
            }
        }
        __syncthreads();
        s[w][lane] = v;
        __syncthreads();
        // thread b of a column: gate row k0 + b
        if (w < batch) {
            float t1 = 0.0f, t0 = 0.0f;
            for (int q = 0; q < parts; q++) {
                t1 += s[w * parts + q][lane].x;
                t0 += s[w * parts + q][lane].y;
            }
            v = make_float2(t1, t0);
            if (post && !sp.whole && p.gate) {
                put(p.dgate, (long long)(k0 + w) * p.dgate_pitch + col, sc * (wp * t1 + bp * t0));
                const float g = at(p.gate, (long long)(k0 + w) * p.gate_pitch + col, 1.0f);
                v = make_float2(t1 * g, t0 * g);
            }
        }
        __syncthreads();
        if (w < batch) s[w][lane] = v;
        __syncthreads();
        if (w == 0)
            for (int b = 0; b < batch; b++) {
                g1 += s[b][lane].x;
                g0 += s[b][lane].y;
            }
    }
    if (w != 0) return;
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

template <typename T, int THREADS, int LPR, int NCH, int STAGES, int FILL>
cudaError_t run_forward_as(const FhResidualNormParams& p, cudaStream_t st) {
    static std::atomic<bool> done[64];
    constexpr size_t smem = Ring<T, THREADS, NCH, 2, STAGES>::kBytes;
    const cudaError_t e = allow(k_residual_norm<T, THREADS, LPR, NCH, STAGES, FILL>, smem, done);
    if (e != cudaSuccess) return e;
    constexpr int RPC = THREADS / LPR;
    const long long want = (p.m + RPC - 1) / RPC;
    const int grid = (int)std::min<long long>(want, (long long)kSms * (kForwardThreads / THREADS));
    return fhk::launch(k_residual_norm<T, THREADS, LPR, NCH, STAGES, FILL>, dim3(grid), dim3(THREADS), smem, st, p,
                       (unsigned)(p.gate ? p.m / p.gates : p.m));
}
template <typename T, int THREADS, int LPR, int NCH, int STAGES>
cudaError_t run_forward(const FhResidualNormParams& p, cudaStream_t st) {
    if (p.c == 8 * LPR * NCH) return run_forward_as<T, THREADS, LPR, NCH, STAGES, kFull>(p, st);
    return p.c % 8 ? run_forward_as<T, THREADS, LPR, NCH, STAGES, kAny>(p, st)
                   : run_forward_as<T, THREADS, LPR, NCH, STAGES, kWholeChunks>(p, st);
}

// Threads a row, chunks a thread and rows in the ring, by the channels alone. A row ahead or two is enough, and more reads in
// flight beside the writes are slower: 16384 x 4096 90 us with 2 rows in the ring, 98 with 3, 99 with 4. Two tiers want a
// third row all the same (16384 x 1536 35.7 us, 40.6 with 2; 4096 x 8192 45.4 and 48.6).
template <typename T>
cudaError_t forward(const FhResidualNormParams& p, cudaStream_t st) {
    const int c8 = (p.c + 7) / 8;
    if (c8 <= 8) return run_forward<T, 256, 8, 1, 3>(p, st);
    if (c8 <= 16) return run_forward<T, 256, 16, 1, 3>(p, st);
    if (c8 <= 32) return run_forward<T, 256, 32, 1, 3>(p, st);
    if (c8 <= 64) return run_forward<T, 256, 32, 2, 2>(p, st);
    if (c8 <= 128) return run_forward<T, 128, 128, 1, 3>(p, st);
    if (c8 <= 256) return run_forward<T, 128, 128, 2, 3>(p, st);
    if (c8 <= 512) return run_forward<T, 256, 256, 2, 2>(p, st);
    return run_forward<T, 512, 512, 2, 3>(p, st);
}

// Slices and runs are whole numbers, so gate rows just past a divisor of the CTAs leave up to half of them without work (above 2048
// channels 75 and 149 gate rows, at 1025 to 2048 or up to 256 channels 150 and 297).
Split split_of(long long m, int c, int gates, bool gate) {
    Split s{};
    s.groups = gate ? gates : 1;
    s.len = m / s.groups;
    // as many CTAs as are resident at once: kGradThreads threads per SM in CTAs of 64 to 512 (grad())
    const int target = kSms * (c > 2048 ? 1 : c > 1024 || c <= 256 ? 2 : c > 512 ? 4 : 8);
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

template <typename T, int THREADS, int LPR, int NCH, int STAGES, bool WHOLE, int FILL, bool ZEROTH>
cudaError_t run_grad_as(const FhResidualNormGradParams& p, const Split& sp, cudaStream_t st) {
    static std::atomic<bool> done[64];
    constexpr size_t smem = Ring<T, THREADS, NCH, 4, STAGES>::kBytes +
                            (NCH > 1 ? NCH * (ZEROTH ? 3 : 1) * Kept<THREADS>::kChunkBytes : 0);
    const cudaError_t e = allow(k_residual_norm_grad<T, THREADS, LPR, NCH, STAGES, WHOLE, FILL, ZEROTH>, smem, done);
    if (e != cudaSuccess) return e;
    return fhk::launch(k_residual_norm_grad<T, THREADS, LPR, NCH, STAGES, WHOLE, FILL, ZEROTH>, dim3(sp.ctas), dim3(THREADS), smem, st, p, sp,
                       static_cast<float*>(p.scratch));
}
template <typename T, int THREADS, int LPR, int NCH, int STAGES>
cudaError_t run_grad(const FhResidualNormGradParams& p, const Split& sp, cudaStream_t st) {
    if (sp.whole) return run_grad_as<T, THREADS, LPR, NCH, STAGES, true, kAny, true>(p, sp, st);
    const int fill = p.c == 8 * LPR * NCH ? kFull : p.c % 8 ? kAny : kWholeChunks;
    if (sp.zeroth)
        return fill == kFull  ? run_grad_as<T, THREADS, LPR, NCH, STAGES, false, kFull, true>(p, sp, st)
               : fill == kAny ? run_grad_as<T, THREADS, LPR, NCH, STAGES, false, kAny, true>(p, sp, st)
                              : run_grad_as<T, THREADS, LPR, NCH, STAGES, false, kWholeChunks, true>(p, sp, st);
    return fill == kFull  ? run_grad_as<T, THREADS, LPR, NCH, STAGES, false, kFull, false>(p, sp, st)
           : fill == kAny ? run_grad_as<T, THREADS, LPR, NCH, STAGES, false, kAny, false>(p, sp, st)
                          : run_grad_as<T, THREADS, LPR, NCH, STAGES, false, kWholeChunks, false>(p, sp, st);
}

// One chunk a thread up to 4096 channels, beside its four column sums. A third row in the ring costs 4 % up to 256
// channels (60,000 x 200 with biases 52.6 us, 54.8 with it) and gains 2 % above 512 (16384 x 2048 with its forward 139.5 us,
// 136.6 with it).
template <typename T>
cudaError_t grad(const FhResidualNormGradParams& p, const Split& sp, cudaStream_t st) {
    const int c8 = (p.c + 7) / 8;
    cudaError_t e;
    if (c8 <= 8) e = run_grad<T, 256, 8, 1, 2>(p, sp, st);
    else if (c8 <= 16) e = run_grad<T, 256, 16, 1, 2>(p, sp, st);
    else if (c8 <= 32) e = run_grad<T, 256, 32, 1, 2>(p, sp, st);
    else if (c8 <= 64) e = run_grad<T, 64, 64, 1, 2>(p, sp, st);
    else if (c8 <= 128) e = run_grad<T, 128, 128, 1, 3>(p, sp, st);
    else if (c8 <= 256) e = run_grad<T, 256, 256, 1, 3>(p, sp, st);
    else if (c8 <= 512) e = run_grad<T, 512, 512, 1, 3>(p, sp, st);
    else e = run_grad<T, 512, 512, 2, 2>(p, sp, st);
    if (e != cudaSuccess) return e;
    const bool post = p.f && (p.dgate || p.dscale || p.dw_post || p.db_post), pre = p.dw_pre || p.db_pre;
    if (!post && !pre) return cudaSuccess;
    fhk::PdlScope pdl(true);  // it waits for the kernel above
    return fhk::launch(k_residual_norm_params<T>, dim3((p.c + 15) / 16, 2), dim3(1024), 0, st, p, sp,
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
    Split sp = split_of(p->m, p->c, p->gates, p->gate != nullptr);
    sp.zeroth = sp.whole || p->b_post || p->db_post || p->db_pre;
    return (int)(p->dtype == FH_F16 ? grad<__half>(*p, sp, st) : grad<__nv_bfloat16>(*p, sp, st));
}
