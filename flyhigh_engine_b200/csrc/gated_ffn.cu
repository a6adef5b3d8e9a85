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
// jobs of one persistent launch, with the biases' gradients beside them), and where K was split one more that adds the
// parts. Each waits for the one before on the device (programmatic dependent launch). Few rows (k_rows) and feature maps
// of few channels (gated_ffn_map.cuh) have forms of their own.
//
// At 8192 rows of 2048 -> 8192 -> 2048 in bf16 the first launch takes 336 us with the tensor pipe active 93 % of the time
// (1,636 TFLOP/s), the second 203 us (72 %: 256 tiles in four turns of 74 CTA pairs); of a training step's gradient da takes
// 267 us (54 %, at 3.8 TB/s of g, u and their gradients) and the four products after it 975 us (84 %).
//
// What is rounded to 16 bits is what the next product takes as its operand: a, dg and du (a product of 32-bit operands would be of
// tf32, at half the rate and twice the bytes). Everything else, g and u among it, stays in 32.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "fh_device.cuh"
#include "ffn_parts.cuh"
#include "fh_kernels.h"
#include "gated_ffn_map.cuh"
#include "launch.h"

namespace {

enum Tail { PLAIN, GLU, GLU_GRAD, GLU_AGAIN };
constexpr int kGroupM = 8;  // tiles of rows that are walked together, so that their operands stay in L2

// n / d for n < 2^31 by a multiplication: with 2^s >= d > 2^(s - 1) and mul = ceil(2^(31 + s) / d), which is below 2^32, the
// product's error stays under n / 2^31 of a step, so its upper bits are the quotient (Granlund and Montgomery)
struct Divider {
    unsigned mul, shift, d;
    Divider() = default;
    __host__ explicit Divider(unsigned by) : d(by) {
        unsigned s_ = 0;
        while ((1ull << s_) < by) s_++;
        shift = s_;
        mul = (unsigned)(((1ull << (31 + s_)) + by - 1) / by);
    }
    __device__ __forceinline__ unsigned div(unsigned n) const { return (unsigned)(((unsigned long long)n * mul) >> (31 + shift)); }
};

// One product of a launch: out[m][n] = tail(sum over the terms of A[t] B[t]^T). GLU: A[0] with B[0] (gate) and B[1] (up).
// GLU_AGAIN: A[0] = dy with B[0] = w_down, and A[1] = x with B[1] = gate and x[2] = up, beside each other: the gradient of
// the activation with g and u formed again instead of read.
struct alignas(64) Job {
    CUtensorMap a[2], b[2], o;     // o: out, in boxes of the tails
    int mn_a, mn_b;                // the operand is MN-major
    int kb[2];                     // 64-deep K blocks of the terms
    int m, n;                      // output extents
    int tiles_m, tiles_n, splits;  // tiles, and the parts of K that different CTAs sum
    int first;                     // its first work item
    Divider by_tiles, by_group;    // tiles_m * tiles_n, kGroupM * tiles_n
    void* out;
    long long pitch;
    const void *bias0, *bias1;  // by column, or NULL
    float* part;                // splits > 1: [split][m][n8] sums in place of out
    void* sums;                 // [m] the rows' sums of A (a bias's gradient), or NULL
    float* sums_part;           // splits > 1: [split][m8] in its place
};
constexpr int kJobs = 4;
struct Work {
    Job job[kJobs];
    CUtensorMap x[3];  // GLU: where g and u are kept (keep); GLU_GRAD: du out, g and u in; GLU_AGAIN: du and a out, w_up
    void* out[2];      // the same outputs
    int jobs, items, bn, stages, act, keep;
    int sums;  // some job's rows are summed: A times a tile of ones, one matrix instruction of 16 columns beside each
    int extra;  // bytes that a stage's barrier expects beyond its copies (0, or a test's)
    long long limit;
};

constexpr int kEpiWarps = 8;
constexpr int kThreads = (kEpiWarps + 2) * 32;
constexpr int kStageA = 128 * 128;  // 128 rows of 64 elements
constexpr int kMaxStages = 8;
// shared memory: the operand ring, then each warp's staging tiles. Four of them are two groups of 64 columns in turn; the tails
// that keep or read g and u in f32, or leave dg, du and a, take six.
constexpr int kOperands = 229376;
constexpr int tail_tiles(bool six) { return six ? 6 : 4; }
constexpr int ring_bytes(bool six) { return kOperands - kEpiWarps * tail_tiles(six) * kTile; }
constexpr int kAgain = 64;  // GLU_AGAIN: hidden columns of a tile (da, g and u of 64 columns each)
constexpr int kOnes = 2048;  // of the ring: 16 rows of ones
constexpr int kBars = 512;
constexpr int kSmem = 1024 + kOperands + kBars;

struct Item {
    const Job* j;
    int tm, tn, split, k0, k1;
};
__device__ __forceinline__ Item item_of(const Work& w, int i) {
    int n = 0;
    while (n + 1 < w.jobs && i >= w.job[n + 1].first) n++;
    const Job& j = w.job[n];
    i -= j.first;
    Item t;
    t.j = &j;
    t.split = j.by_tiles.div(i);
    i -= t.split * (int)j.by_tiles.d;
    const int grp = j.by_group.div(i), rows_ = min(kGroupM, j.tiles_m - grp * kGroupM);
    i -= grp * (int)j.by_group.d;
    t.tn = rows_ == kGroupM ? i / kGroupM : i / rows_;
    t.tm = grp * kGroupM + i - t.tn * rows_;
    const int kb = j.kb[0] + j.kb[1];
    t.k0 = 0, t.k1 = kb;
    if (j.splits > 1) {
        t.k0 = (int)((long long)kb * t.split / j.splits);
        t.k1 = (int)((long long)kb * (t.split + 1) / j.splits);
    }
    return t;
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
    // bn: columns of an accumulator; nb: rows of B that this CTA holds
    const int bn = w.bn, nb = TAIL == GLU_AGAIN ? 2 * kAgain : bn / CTAS, stages = w.stages;
    const uint32_t stage_bytes = kStageA + nb * 128;
    const bool keep = TAIL == GLU && w.keep, f32 = keep || TAIL == GLU_GRAD, six = f32 || TAIL == GLU_AGAIN;
    const uint32_t staging = base + ring_bytes(six), bars = base + kOperands;
    const uint32_t full = bars, empty = bars + 8 * kMaxStages, tfull = bars + 16 * kMaxStages, tempty = tfull + 16,
                   slot = tempty + 16;
    const uint32_t ones = base + ring_bytes(six) - kOnes;
    const uint32_t cols = TAIL == GLU_AGAIN ? 512 : TAIL == PLAIN && w.sums ? 4 * bn : 2 * bn;  // sums: 32 beside each 2 bn

    if (warp == 8 && lane == 0) {
        for (int s = 0; s < stages; s++) {
            bar_init(full + 8 * s, 1);
            bar_init(empty + 8 * s, 1);
        }
        for (int b = 0; b < 2; b++) {
            bar_init(tfull + 8 * b, 1);
            bar_init(tempty + 8 * b, kEpiWarps * CTAS);
        }
        for (int q = 0; q < 2 * kEpiWarps; q++) bar_init(bars + 256 + 8 * q, 1);
        bar_init_fence();
    }
    if (TAIL == PLAIN && w.sums && warp < 4) {  // whatever the order of a tile of ones
        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};\n" ::"r"(ones + 16 * threadIdx.x),
                     "r"(std::is_same<T, __half>::value ? 0x3c003c00u : 0x3f803f80u)
                     : "memory");
        fence_async();
    }
    if (warp == 9) tmem_alloc<CTAS>(slot, cols);
    fence_before();
    if (CTAS == 2) cluster_sync();
    else __syncthreads();
    fence_after();
    uint32_t tbase;
    asm volatile("ld.shared.b32 %0, [%1];\n" : "=r"(tbase) : "r"(slot));
    tbase = uniform(tbase);
    pdl_wait();
    pdl_trigger();

    const int first = blockIdx.x / CTAS, step = gridDim.x / CTAS;
    // the matrix instructions are issued by the pair's first CTA
    auto free_accumulators = [&](uint32_t bar) {
        if (CTAS == 1 || rank == 0) bar_arrive(bar);
        else bar_arrive_cluster(map_rank(bar, 0));
    };
    bool ok = true;
    auto wait = [&](uint32_t bar, uint32_t parity) {  // by whole warps
        if (ok) ok = __all_sync(0xffffffffu, bar_wait(bar, parity, w.limit, &g_ffn_timeouts));
        return ok;
    };
    if (warp == 8) {
        const bool leader = elected();
        int s = 0;
        uint32_t ph = 1;  // the ring starts empty
        for (int i = first; ok && i < w.items; i += step) {
            const Item t = item_of(w, i);
            const Job& j = *t.j;
            const int row = t.tm * 128 * CTAS + (int)rank * 128;
            const int kb0 = j.kb[0];
            const bool mn_a = j.mn_a, mn_b = j.mn_b;
            for (int k = t.k0; k < t.k1; k++) {
                if (!wait(empty + 8 * s, ph)) break;
                const int term = TAIL != GLU && k >= kb0, kk = (k - (term ? kb0 : 0)) * BK;
                const uint32_t bar = CTAS == 2 ? map_rank(full + 8 * s, 0) : full + 8 * s;
                const uint32_t da = base + s * stage_bytes, db = da + kStageA;
                const CUtensorMap* ma = &j.a[term];
                const CUtensorMap* mb = &j.b[TAIL == GLU && CTAS == 2 ? rank : term];
                if (leader) {
                    if (rank == 0) bar_expect(full + 8 * s, CTAS * (TAIL == GLU_AGAIN && !term ? stage_bytes - kAgain * 128 : stage_bytes) + w.extra);
                    if (mn_a) {
                        tensor_load<CTAS>(da, ma, row, kk, bar);
                        tensor_load<CTAS>(da + 8192, ma, row + 64, kk, bar);
                    } else {
                        tensor_load<CTAS>(da, ma, kk, row, bar);
                    }
                    if (TAIL == GLU_AGAIN) {
                        const int c = t.tn * kAgain;
                        tensor_load<CTAS>(db, mb, term ? kk : c, term ? c : kk, bar);
                        if (term) tensor_load<CTAS>(db + kAgain * 128, &w.x[2], kk, c, bar);
                    } else if (TAIL == GLU) {
                        const int c = t.tn * (bn / 2);
                        tensor_load<CTAS>(db, mb, kk, c, bar);
                        if (CTAS == 1) tensor_load<CTAS>(db + (bn / 2) * 128, &j.b[1], kk, c, bar);
                    } else {
                        const int c = t.tn * bn + (int)rank * nb;
                        if (mn_b)
                            for (int q = 0; q < nb / 64; q++) tensor_load<CTAS>(db + q * 8192, mb, c + 64 * q, kk, bar);
                        else
                            tensor_load<CTAS>(db, mb, kk, c, bar);
                    }
                }
                __syncwarp();
                if (++s == stages) s = 0, ph ^= 1;
            }
        }
    } else if (warp == 9) {
        if (rank == 0) {
            const bool leader = elected();
            int s = 0, n = 0;
            uint32_t ph = 0;
            for (int i = first; ok && i < w.items; i += step, n++) {
                const Item t = item_of(w, i);
                const Job& j = *t.j;
                const int b = n & 1;
                const uint32_t d = tbase + b * bn;
                const uint32_t idesc = instr_desc(!std::is_same<T, __half>::value, j.mn_a, j.mn_b, 128 * CTAS, bn);
                // one K step of 16: 32 bytes along a K-major tile's rows, two 8-k groups of an MN-major one
                const uint32_t sa = j.mn_a ? 2048 >> 4 : 32 >> 4, sb = j.mn_b ? 2048 >> 4 : 32 >> 4;
                const bool sums = TAIL == PLAIN && j.sums && t.tn == 0;
                const uint32_t idsum = instr_desc(!std::is_same<T, __half>::value, j.mn_a, false, 128 * CTAS, 16 * CTAS);
                if (!wait(tempty + 8 * b, ((n >> 1) & 1) ^ 1)) break;
                fence_after();
                for (int k = t.k0; k < t.k1; k++) {
                    if (!wait(full + 8 * s, ph)) break;
                    fence_after();
                    const uint32_t da = base + s * stage_bytes;
                    const uint64_t ad = tile_desc(da, 8192), bd = tile_desc(da + kStageA, 8192);
                    if (TAIL == GLU_AGAIN) {  // da (w_down is MN-major), then g and u side by side
                        const bool again = k >= j.kb[0];
                        const uint32_t id = instr_desc(!std::is_same<T, __half>::value, false, !again, 128, again ? 2 * kAgain : kAgain);
                        const uint32_t to = again ? d + kAgain : d, step_b = again ? 32 >> 4 : 2048 >> 4;
                        if (leader) {
#pragma unroll
                            for (int q = 0; q < 4; q++)
                                mma<CTAS>(to, ad + q * (32 >> 4), bd + q * step_b, id, (k > (again ? j.kb[0] : 0) || q > 0) ? 1u : 0u);
                            commit<CTAS>(empty + 8 * s);
                        }
                    } else if (leader) {
#pragma unroll
                        for (int q = 0; q < 4; q++) mma<CTAS>(d, ad + q * sa, bd + q * sb, idesc, (k > t.k0 || q > 0) ? 1u : 0u);
                        if (sums)
#pragma unroll
                            for (int q = 0; q < 4; q++)
                                mma<CTAS>(tbase + 2 * bn + 32 * b, ad + q * sa, tile_desc(ones, 0), idsum, (k > t.k0 || q > 0) ? 1u : 0u);
                        commit<CTAS>(empty + 8 * s);
                    }
                    if (++s == stages) s = 0, ph ^= 1;
                }
                if (ok && leader) commit<CTAS>(tfull + 8 * b);
            }
        }
    } else {
        // the tails: this warp's 32 rows and half of the tile's columns (all of a 32-wide tile for the first half), in groups
        // of 64 (32 where g and u are kept or read) that pass through staging tiles of 32 x 32 (f32: 32 x 16), which tensor
        // copies store, clipped at the output's edges. g and u are kept in f32: rounded to 16 bits they would put two more
        // roundings of that size into every gradient behind them (1.8 against 1.4 times the error of one rounding).
        const int group = six ? 32 : 64;
        const int q = warp & 3, half = warp >> 2;
        const int width = TAIL == GLU ? bn / 2 : TAIL == GLU_AGAIN ? kAgain : bn, span = max(32, width / 2);
        const int lo = half * span, hi = min(width, lo + span);
        const uint32_t tiles = staging + warp * tail_tiles(six) * kTile, gbar = bars + 256 + 16 * warp;
        int n = 0, turn = 0;  // turn: the pair of four tiles that is next
        uint32_t gph = 0;
        for (int i = first; i < w.items; i += step, n++) {
            const Item t = item_of(w, i);
            const Job* j = t.j;
            const int b = n & 1, m = j->m, cols_ = j->n, col = t.tn * width;
            const int row = t.tm * 128 * CTAS + (int)rank * 128 + q * 32;
            float* part = j->part;
            const void *bias0 = part ? nullptr : j->bias0, *bias1 = j->bias1;
            const bool ragged = cols_ & 7, biased = bias0 || bias1;
            auto live = [&](int c0) { return row < m && c0 < hi && col + c0 < cols_; };
            // GLU_GRAD: g and u of 16 columns into tiles 2 h and 2 h + 1; they are on their way a group ahead
            auto fetch = [&](int c0, int h) {
                if (!live(c0) || lane != 0) return;
                const uint32_t bar = gbar + 8 * h, dst = tiles + 2 * h * kTile;
                bar_expect(bar, 2 * kTile);
                tensor_load<1>(dst, &w.x[1], col + c0, row, bar);
                tensor_load<1>(dst + kTile, &w.x[2], col + c0, row, bar);
            };
            if (TAIL == GLU_GRAD) {
                fetch(lo, 0);
                fetch(lo + 16, 1);
                __syncwarp();
            }
            if (!wait(tfull + 8 * b, (n >> 1) & 1)) break;
            fence_after();
            const uint32_t acc = tbase + ((uint32_t)(q * 32) << 16) + b * bn;
            if (TAIL == PLAIN && j->sums && t.tn == 0 && half == 0) {
                uint32_t v;
                load1(tbase + ((uint32_t)(q * 32) << 16) + 2 * bn + 32 * b, v);
                wait_ld();
                if (row + lane < m) {
                    if (part) j->sums_part[(long long)t.split * ((m + 7) & ~7) + row + lane] = __uint_as_float(v);
                    else static_cast<T*>(j->sums)[row + lane] = Elem<T>::from(__uint_as_float(v));
                }
                __syncwarp();
            }
            for (int c0 = lo; c0 < hi; c0 += group) {
                const bool alive = live(c0);
                // this group's tiles: a pair of 16-bit ones in turn (three: dg, du, a); or a, g (2), u (2); or dg and du behind
                // g's and u's four
                const uint32_t dst = keep ? tiles : TAIL == GLU_GRAD ? tiles + 4 * kTile : tiles + (TAIL == GLU_AGAIN ? 3 : 2) * (turn & 1) * kTile;
                if (lane == 0) {  // what they held has been read
                    if (f32) stores_read<0>();
                    else stores_read<1>();
                }
                __syncwarp();
                const int subs = min(group, hi - c0) / 32;
                if constexpr (TAIL == GLU_AGAIN) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int cs = c0 + 16 * h;
                        uint32_t r0[16], r1[16], r2[16], q0[8], q1[8];
                        load16(acc + cs, r0);
                        load16(acc + kAgain + cs, r1);
                        load16(acc + 2 * kAgain + cs, r2);
                        if (biased) {
                            load_bias<T>(bias0, col + cs, cols_, q0);
                            load_bias<T>(bias1, col + cs, cols_, q1);
                            __syncwarp();
                        }
                        wait_ld();
                        if (h == 1) {
                            fence_before();
                            __syncwarp();
                            if (lane == 0) free_accumulators(tempty + 8 * b);
                        }
                        float2 v[8], g[8], u[8], a[8];
                        pairs(r0, v);
                        pairs(r1, g);
                        pairs(r2, u);
                        if (biased) {
                            add_bias<T>(q0, g);
                            add_bias<T>(q1, u);
                        }
                        switch (w.act) {
                            case FH_ACT_SILU: glu_grad16<FH_ACT_SILU>(v, g, u, a); break;
                            case FH_ACT_GELU: glu_grad16<FH_ACT_GELU>(v, g, u, a); break;
                            case FH_ACT_GELU_TANH: glu_grad16<FH_ACT_GELU_TANH>(v, g, u, a); break;
                            case FH_ACT_RELU: glu_grad16<FH_ACT_RELU>(v, g, u, a); break;
                            default: glu_grad16<FH_ACT_SIGMOID>(v, g, u, a); break;
                        }
                        tile_put<T>(dst, lane, h, g);
                        tile_put<T>(dst + kTile, lane, h, u);
                        tile_put<T>(dst + 2 * kTile, lane, h, a);
                        __syncwarp();
                    }
                }
                for (int sub = 0; TAIL != GLU_AGAIN && sub < subs; sub++) {
                    const int cs = c0 + 32 * sub;
                    uint32_t r0[32], r1[TAIL == GLU ? 32 : 1], q0[16], q1[16];
                    load32(acc + cs, r0);
                    if constexpr (TAIL == GLU) load32(acc + bn / 2 + cs, r1);
                    if (TAIL != GLU_GRAD && biased) {
                        load_bias<T>(bias0, col + cs, cols_, q0);
                        if (TAIL == GLU) load_bias<T>(bias1, col + cs, cols_, q1);
                        __syncwarp();
                    }
                    wait_ld();
                    if (cs + 32 >= hi) {  // the accumulators have been read
                        fence_before();
                        __syncwarp();
                        if (lane == 0) free_accumulators(tempty + 8 * b);
                    }
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        float2 v[8], g[8], u[8];
                        if constexpr (TAIL == GLU) {
                            pairs(r0 + 16 * h, g);
                            pairs(r1 + 16 * h, u);
                            if (biased) {
                                add_bias<T>(q0 + 8 * h, g);
                                add_bias<T>(q1 + 8 * h, u);
                            }
                            switch (w.act) {
                                case FH_ACT_SILU: glu16<FH_ACT_SILU>(g, u, v); break;
                                case FH_ACT_GELU: glu16<FH_ACT_GELU>(g, u, v); break;
                                case FH_ACT_GELU_TANH: glu16<FH_ACT_GELU_TANH>(g, u, v); break;
                                case FH_ACT_RELU: glu16<FH_ACT_RELU>(g, u, v); break;
                                default: glu16<FH_ACT_SIGMOID>(g, u, v); break;
                            }
                            tile_put<T>(dst + sub * kTile, lane, h, v);
                            if (keep) {
                                tile_put32(dst + (1 + h) * kTile, lane, g);
                                tile_put32(dst + (3 + h) * kTile, lane, u);
                            }
                        } else if constexpr (TAIL == GLU_GRAD) {
                            pairs(r0 + 16 * h, v);
                            if (live(cs + 16 * h)) {
                                wait(gbar + 8 * h, (gph >> h) & 1);
                                gph ^= 1u << h;
                            }
                            if (!ok) break;
                            tile_get32(tiles + 2 * h * kTile, lane, g);
                            tile_get32(tiles + (2 * h + 1) * kTile, lane, u);
                            switch (w.act) {
                                case FH_ACT_SILU: glu_grad16<FH_ACT_SILU>(v, g, u, v); break;
                                case FH_ACT_GELU: glu_grad16<FH_ACT_GELU>(v, g, u, v); break;
                                case FH_ACT_GELU_TANH: glu_grad16<FH_ACT_GELU_TANH>(v, g, u, v); break;
                                case FH_ACT_RELU: glu_grad16<FH_ACT_RELU>(v, g, u, v); break;
                                default: glu_grad16<FH_ACT_SIGMOID>(v, g, u, v); break;
                            }
                            tile_put<T>(dst, lane, h, g);
                            tile_put<T>(dst + kTile, lane, h, u);
                            // The copy that takes the tiles' place next is ordered behind this warp's reads by nothing but
                            // these: every lane's values have arrived (dg and du, stored above, are formed from all of them),
                            // and the fence keeps reads before it from copies after it. Issued right after the loads, behind a
                            // __syncwarp alone, the copy overtook them where memory was busy: g of the next group in some lanes.
                            fence_async();
                            __syncwarp();
                            fetch(cs + 32 + 16 * h, h);
                            __syncwarp();
                        } else {
                            pairs(r0 + 16 * h, v);
                            if (part) {
                                const int c = col + cs + 16 * h, valid = cols_ - c;
                                if (row + lane < m) {
                                    const long long n8 = (cols_ + 7) & ~7;
                                    float4* o = reinterpret_cast<float4*>(part + ((long long)t.split * m + row + lane) * n8 + c);
#pragma unroll
                                    for (int e = 0; e < 4; e++)  // columns up to n8 are the scratch's own
                                        if (4 * e < valid) o[e] = make_float4(v[2 * e].x, v[2 * e].y, v[2 * e + 1].x, v[2 * e + 1].y);
                                }
                                __syncwarp();
                            } else {
                                if (biased) add_bias<T>(q0 + 8 * h, v);
                                tile_put<T>(dst + sub * kTile, lane, h, v);
                            }
                        }
                    }
                }
                if (!ok) break;
                if (!alive || (TAIL == PLAIN && part)) continue;
                fence_async();
                __syncwarp();
                if (ragged && col + c0 + group > cols_) {  // the columns end inside a 16-byte piece
                    for (int sub = 0; sub < subs && col + c0 + 32 * sub < cols_; sub++) {
                        const long long at = (long long)(row + lane) * j->pitch + col + c0 + 32 * sub;
                        const int valid = min(32, cols_ - col - c0 - 32 * sub);
                        if (row + lane >= m) continue;
                        tile_out<T>(dst + sub * kTile, lane, static_cast<T*>(j->out) + at, valid);
                        for (int h = 0; keep && 16 * h < valid; h++) {
                            tile_out32(dst + (1 + h) * kTile, lane, static_cast<float*>(w.out[0]) + at + 16 * h, min(16, valid - 16 * h));
                            tile_out32(dst + (3 + h) * kTile, lane, static_cast<float*>(w.out[1]) + at + 16 * h, min(16, valid - 16 * h));
                        }
                        if (TAIL == GLU_GRAD || TAIL == GLU_AGAIN) tile_out<T>(dst + kTile, lane, static_cast<T*>(w.out[0]) + at, valid);
                        if (TAIL == GLU_AGAIN) tile_out<T>(dst + 2 * kTile, lane, static_cast<T*>(w.out[1]) + at, valid);
                    }
                    fence_async();
                    __syncwarp();
                    if (lane == 0) stores_commit();  // a group of no stores: the count of those before stays right
                } else if (lane == 0) {
                    for (int sub = 0; sub < subs && col + c0 + 32 * sub < cols_; sub++)
                        tensor_store(&j->o, col + c0 + 32 * sub, row, dst + sub * kTile);
                    for (int h = 0; keep && h < 2 && col + c0 + 16 * h < cols_; h++) {
                        tensor_store(&w.x[0], col + c0 + 16 * h, row, dst + (1 + h) * kTile);
                        tensor_store(&w.x[1], col + c0 + 16 * h, row, dst + (3 + h) * kTile);
                    }
                    if (TAIL == GLU_GRAD || TAIL == GLU_AGAIN) tensor_store(&w.x[0], col + c0, row, dst + kTile);
                    if (TAIL == GLU_AGAIN) tensor_store(&w.x[1], col + c0, row, dst + 2 * kTile);
                    stores_commit();
                }
                turn++;
            }
            if (!ok) break;
            // a half without columns of a narrow tile
            if (lo >= hi) {
                fence_before();
                __syncwarp();
                if (lane == 0) free_accumulators(tempty + 8 * b);
            }
        }
        if (lane == 0) stores_done();
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

// ---- few rows ----
//
// With up to 32 rows the weights are what has to be read, once, at HBM's rate; a 128-row tile would leave its matrix pipe idle
// and the grid short of CTAs. Here the weights' rows are the 16 rows of mma.m16n8k16 and x's rows its 8 columns (NT of them
// side by side), so a CTA of 8 warps produces 16 output channels for all rows. Its warps take 32-wide steps of K in turn and
// are added in shared memory; where the channels alone would not fill the GPU a cluster's CTAs share K and add over
// distributed shared memory. Operands go from global memory to fragments: a thread's four k positions of two MMAs are
// 8 consecutive elements of its row (the same order of k for both operands), one 16-byte load each.
template <typename T>
struct RowsArgs {
    const T *x, *w0, *w1;  // [m][k], [n][k]
    long long x_pitch, w0_pitch, w1_pitch;
    const T *bias0, *bias1;
    T* out;
    float *g, *u;
    long long pitch;
    int m, n, k, act, share;  // share: CTAs of a cluster
};
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                                 uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                        uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 8 elements of a row from k on, 0 past its end (the last step of K). The 16 bytes that hold an element of the row are read
// whole (they lie inside its pitch) and what is not the row's is masked.
template <typename T>
__device__ __forceinline__ uint4 load_k(const T* row, int k, int end) {
    uint4 q = make_uint4(0, 0, 0, 0);
    if (k >= end) return q;
    q = *reinterpret_cast<const uint4*>(row + k);
    auto cut = [&](uint32_t w, int first) { return k + first + 1 < end ? w : k + first < end ? w & 0xffffu : 0u; };
    return make_uint4(cut(q.x, 0), cut(q.y, 2), cut(q.z, 4), cut(q.w, 6));
}
// 16 bytes of a weight: read once, so not kept in L1
template <typename T>
__device__ __forceinline__ uint4 load_once(const T* p) {
    uint4 q;
    asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w) : "l"(p));
    return q;
}
__device__ __forceinline__ float act_by(int act, float g) {
    const float2 v = pair(g);
    switch (act) {
        case FH_ACT_SILU: return act_of<FH_ACT_SILU>(v).x;
        case FH_ACT_GELU: return act_of<FH_ACT_GELU>(v).x;
        case FH_ACT_GELU_TANH: return act_of<FH_ACT_GELU_TANH>(v).x;
        case FH_ACT_RELU: return act_of<FH_ACT_RELU>(v).x;
        default: return act_of<FH_ACT_SIGMOID>(v).x;
    }
}

template <typename T, int NT, bool GATED>
__global__ void __launch_bounds__(256, 2) k_rows(const RowsArgs<T> p) {
    constexpr int NW = GATED ? 2 : 1, COLS = 8 * NT, UNROLL = NT == 1 ? 4 : 2;
    __shared__ float part[4][NW][COLS][17];  // [warp % 4][matrix][row of x][channel]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int tile = blockIdx.x / p.share, rank = blockIdx.x - tile * p.share;
    const int steps = (p.k + 31) / 32, lo = steps * rank / p.share, hi = steps * (rank + 1) / p.share, inside = min(hi, p.k / 32);
    // a row that is not there reads the last one: its results go nowhere
    const T* w[NW][2];
    const T* x[NT];
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const long long c = min(tile * 16 + g + 8 * e, p.n - 1);
        w[0][e] = p.w0 + c * p.w0_pitch;
        if (GATED) w[NW - 1][e] = p.w1 + c * p.w1_pitch;
    }
#pragma unroll
    for (int i = 0; i < NT; i++) x[i] = p.x + (long long)min(8 * i + g, p.m - 1) * p.x_pitch;
    float acc[NW][NT][4] = {};
    uint4 a[UNROLL][NW][2], b[UNROLL][NT];
    // step s: one of this CTA's, wholly inside K; the last one may not be, and behind hi there is nothing
    auto load_weights = [&](int s0) {
        const int k0 = s0 * 32 + 8 * t;
#pragma unroll
        for (int q = 0; q < UNROLL; q++) {
            const int s = s0 + 8 * q;
#pragma unroll
            for (int i = 0; i < NW; i++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    if (s < inside) a[q][i][e] = load_once(w[i][e] + k0 + 256 * q);
                    else a[q][i][e] = s < hi ? load_k(w[i][e], k0 + 256 * q, p.k) : make_uint4(0, 0, 0, 0);
                }
        }
    };
    auto load_x = [&](int s0) {
        const int k0 = s0 * 32 + 8 * t;
#pragma unroll
        for (int q = 0; q < UNROLL; q++) {
            const int s = s0 + 8 * q;
#pragma unroll
            for (int i = 0; i < NT; i++) {
                if (s < inside) b[q][i] = *reinterpret_cast<const uint4*>(x[i] + k0 + 256 * q);
                else b[q][i] = s < hi ? load_k(x[i], k0 + 256 * q, p.k) : make_uint4(0, 0, 0, 0);
            }
        }
    };
    // the weights are no output of the kernel before: they are on their way while it ends
    load_weights(lo + warp);
    pdl_wait();
    pdl_trigger();
    for (int s0 = lo + warp; s0 < hi; s0 += 8 * UNROLL) {
        load_x(s0);
#pragma unroll
        for (int q = 0; q < UNROLL; q++)
#pragma unroll
            for (int i = 0; i < NW; i++)
#pragma unroll
                for (int c = 0; c < NT; c++) {
                    mma16816<T>(acc[i][c], a[q][i][0].x, a[q][i][1].x, a[q][i][0].y, a[q][i][1].y, b[q][c].x, b[q][c].y);
                    mma16816<T>(acc[i][c], a[q][i][0].z, a[q][i][1].z, a[q][i][0].w, a[q][i][1].w, b[q][c].z, b[q][c].w);
                }
        if (s0 + 8 * UNROLL < hi) load_weights(s0 + 8 * UNROLL);
    }
    for (int round = 1; round >= 0; round--) {  // the upper four warps' sums, then the lower four's added to them
        if (warp / 4 == round)
#pragma unroll
            for (int i = 0; i < NW; i++)
#pragma unroll
                for (int c = 0; c < NT; c++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        float& v = part[warp & 3][i][8 * c + 2 * t + (e & 1)][g + 8 * (e >> 1)];
                        v = round ? acc[i][c][e] : v + acc[i][c][e];
                    }
        __syncthreads();
    }
    // the warps' sums in order; in a cluster into the first warp's place, where the other CTAs read them
    auto added = [&](int mat, int r, int c) {
        float v = part[0][mat][r][c];
#pragma unroll
        for (int q = 1; q < 4; q++) v += part[q][mat][r][c];
        return v;
    };
    if (p.share > 1) {
        for (int i = threadIdx.x; i < NW * COLS * 16; i += 256) {
            const int c = i & 15, r = (i >> 4) % COLS, mat = (i >> 4) / COLS;
            part[0][mat][r][c] = added(mat, r, c);
        }
        umma::cluster_sync();
    }
    // each CTA of the cluster finishes a share of the rows
    const int live = min(p.m, COLS), r_lo = live * rank / p.share, r_hi = live * (rank + 1) / p.share;
    for (int i = r_lo * 16 + threadIdx.x; i < r_hi * 16; i += 256) {
        const int c = i & 15, r = i >> 4, col = tile * 16 + c;
        if (col >= p.n) continue;
        float v[NW];
#pragma unroll
        for (int mat = 0; mat < NW; mat++) {
            if (p.share == 1) {
                v[mat] = added(mat, r, c);
                continue;
            }
            const uint32_t at = umma::smem_addr(&part[0][mat][r][c]);
            v[mat] = 0.0f;
            for (int q = 0; q < p.share; q++) {
                float f;
                asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(f) : "r"(umma::map_rank(at, q)) : "memory");
                v[mat] += f;
            }
        }
        if (p.bias0) v[0] += Elem<T>::to(p.bias0[col]);
        const long long at = r * p.pitch + col;
        if (GATED) {
            if (p.bias1) v[NW - 1] += Elem<T>::to(p.bias1[col]);
            p.out[at] = Elem<T>::from(act_by(p.act, v[0]) * v[NW - 1]);
            if (p.g) {
                p.g[at] = v[0];
                p.u[at] = v[NW - 1];
            }
        } else {
            p.out[at] = Elem<T>::from(v[0]);
        }
    }
    if (p.share > 1) umma::cluster_sync();  // the other CTAs may still read this one's sums
}

// Sums over slices: out[r][c] = bias[c] + sum over s of part[s][r][c], for the split products of a launch and for the
// gradients of the biases (one row). 4 columns per thread and 8 threads over the slices, added in order.
struct Sum {
    const float* part;  // [slices][m][n8]
    void* out;
    const void* bias;
    long long pitch, m;
    int n, slices;
    long long first;  // its first group of 4 columns
};
constexpr int kSums = kJobs + 3;  // the products, and three biases
struct Sums {
    Sum s[kSums];
    int n;
    long long total;
};
template <typename T>
__global__ void __launch_bounds__(256) k_sums(const Sums w) {
    __shared__ float4 fold[8][32];
    const int lane = threadIdx.x & 31, way = threadIdx.x >> 5;
    const long long at = (long long)blockIdx.x * 32 + lane;
    int k = 0;
    while (k + 1 < w.n && at >= w.s[k + 1].first) k++;
    const Sum& j = w.s[k];
    const int quads = ((j.n + 7) & ~7) / 4;
    const long long unit = at - j.first, row = unit / quads, slice = j.m * quads;
    const int c = (int)(unit - row * quads) * 4;
    pdl_wait();
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (at < w.total) {
        const float4* p = reinterpret_cast<const float4*>(j.part) + unit;
#pragma unroll 4
        for (int s = way; s < j.slices; s += 8) {
            const float4 t = p[s * slice];
            v.x += t.x, v.y += t.y, v.z += t.z, v.w += t.w;
        }
    }
    fold[way][lane] = v;
    __syncthreads();
    if (way != 0 || at >= w.total) return;
    for (int s = 1; s < 8; s++) {
        const float4 t = fold[s][lane];
        v.x += t.x, v.y += t.y, v.z += t.z, v.w += t.w;
    }
    T* o = static_cast<T*>(j.out) + row * j.pitch + c;
    const float r[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (c + e < j.n) o[e] = Elem<T>::from(r[e] + (j.bias ? Elem<T>::to(static_cast<const T*>(j.bias)[c + e]) : 0.0f));
}

// Column sums of up to three matrices: a CTA sums a slice of the rows of 64 columns (8 threads of 8 columns by 32 rows);
// k_sums adds the slices
struct Columns {
    const void* x;
    long long pitch;
    int n;
    float* part;  // [slices][n8]
};
struct ColumnSums {
    Columns c[3];
    long long m;
    int slices;
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
    Chunk v;
    v.zero();
    if (valid)
#pragma unroll 4
        for (long long i = lo + r; i < hi; i += 32) {
            const Chunk t = load_chunk(static_cast<const T*>(q.x) + i * q.pitch + c, valid);
#pragma unroll
            for (int e = 0; e < 4; e++) v.v[e] = add2(v.v[e], t.v[e]);
        }
#pragma unroll
    for (int e = 0; e < 8; e++) s[r][8 * (threadIdx.x & 7) + e] = v.get(e);
    __syncthreads();
    const int n8 = (q.n + 7) & ~7, col = blockIdx.x * 64 + threadIdx.x;
    if (threadIdx.x < 64 && col < n8) {
        float t = 0.0f;
        for (int i = 0; i < 32; i++) t += s[i][threadIdx.x];
        q.part[(long long)blockIdx.y * n8 + col] = t;
    }
}

// ---- host: tensor maps, the choice of tiles, launches ----

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
    Matrix up;   // GLU_AGAIN
    void* sums;  // of A's rows, with bn <= 128
};

struct Shape {
    int ctas, bn, splits[kJobs];
};

// The tiles of a launch: 256 x 256 or 256 x 128 by a pair of CTAs, or 128 x 128 or 128 x 64 by one; and into how many
// parts each job's K is cut where the tiles leave SMs idle. Chosen by an estimate in SM cycles: a K block of 64 takes the
// larger of the matrix pipe (128 x bn x 16 in bn / 2 cycles, 46 at least) and its operands' way into shared memory (about 56
// bytes per cycle and SM); the tail of an item is hidden by the next item's products, its last one's is not; items go
// round the CTAs, so that more of them than CTAs cost half a longest item at the end; split sums are written and read at
// about 1,600 bytes per cycle and cost another launch of about 8,500 cycles. All jobs' items are cut to a like length: the
// longest K over a few numbers of cuts. Over eight shapes from 300 x 256 -> 1024 to 60,000 x 200 -> 704, forward and gradient
// (11 to 243 us), the choice took 0 to 8 % longer than the best of all kinds and cuts, in one case 21 % (the gradient of
// 3941 x 288 -> 320: 33.2 us where 128 x 64 tiles with four cuts take 27.4).
template <int TAIL>
Shape shape_of(const Product* p, int n) {
    if (TAIL == GLU_AGAIN) {  // 128 x 64 by one CTA
        Shape s{};
        s.ctas = 1, s.bn = 3 * kAgain, s.splits[0] = 1;
        return s;
    }
    static const int kinds[4][2] = {{2, 256}, {2, 128}, {1, 128}, {1, 64}};
    Shape best{};
    double best_t = 1e300;
    long long kb[kJobs], longest_kb = 1;
    for (int i = 0; i < n; i++) {
        kb[i] = (p[i].k + 63) / 64 * p[i].terms;
        longest_kb = std::max(longest_kb, kb[i]);
    }
    for (const auto& kind : kinds) {
        Shape s{};
        s.ctas = kind[0], s.bn = kind[1];
        const int slots = kSms / s.ctas, cols = TAIL == GLU ? s.bn / 2 : s.bn;
        const double per_kb = std::max({2.0 * s.bn, 184.0, (128.0 + s.bn / s.ctas) * 128 / 56});
        const double tail = 1200.0 + s.bn * (TAIL == PLAIN ? 5.0 : TAIL == GLU ? 8.0 : 14.0);
        double tiles[kJobs];
        for (int i = 0; i < n; i++)
            tiles[i] = (double)((p[i].m + 128 * s.ctas - 1) / (128 * s.ctas)) * ((p[i].n + cols - 1) / cols);
        static const int tried[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};
        for (const int cuts : tried) {
            const long long len = (longest_kb + cuts - 1) / cuts;
            if (cuts > 1 && (len < 4 || TAIL != PLAIN)) break;
            double busy = 0, longest = 0, extra = 0, items = 0;
            for (int i = 0; i < n; i++) {
                const int sp = p[i].can_split ? (int)std::max<long long>(1, std::min<long long>(64, kb[i] / len)) : 1;
                s.splits[i] = sp;
                const double item = std::max((double)((kb[i] + sp - 1) / sp) * per_kb, tail);
                items += tiles[i] * sp;
                busy += tiles[i] * sp * item;
                longest = std::max(longest, item);
                if (sp > 1) extra += 8500.0 * (extra == 0) + (double)p[i].m * p[i].n * 8 * sp / 1600;
            }
            const double t = (items <= slots ? longest : busy / slots + 0.5 * longest) + tail + extra;
            if (t < best_t) best_t = t, best = s;
            if (items >= 4.0 * slots && cuts == 1) break;
        }
    }
    return best;
}

size_t product_part_floats(const Product& p, int splits) { return (size_t)splits * (size_t)p.m * (size_t)((p.n + 7) & ~7); }
size_t part_floats(const Product& p, int splits) {
    return splits > 1 ? product_part_floats(p, splits) + (p.sums ? (size_t)splits * (size_t)((p.m + 7) & ~7) : 0) : 0;
}
size_t scratch_floats(const Shape& s, const Product* p, int n) {
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

// the products of one launch; part: scratch_floats, whose sums are added to `sums`
template <typename T, int TAIL, typename P>
cudaError_t products(const Shape& s, const Product* p, int n, const P& call, float* part, Sums* sums, cudaStream_t st) {
    const int dtype = call.dtype;
    Work w;
    w.jobs = n, w.items = 0, w.bn = s.bn, w.act = call.act, w.keep = 0, w.sums = 0, w.extra = call.test_extra_tx;
    w.limit = call.wait_cycles > 0 ? call.wait_cycles : 2000000000ll;
    const int nb = TAIL == GLU_AGAIN ? 2 * kAgain : s.bn / s.ctas;
    bool ones = false;
    for (int i = 0; i < n; i++) ones = ones || p[i].sums;
    w.stages = std::min(kMaxStages, (-(ones ? kOnes : 0) + ring_bytes(TAIL == GLU_GRAD || TAIL == GLU_AGAIN || (TAIL == GLU && p[0].out1))) / (kStageA + nb * 128));
    for (int i = 0; i < n; i++) {
        Job& j = w.job[i];
        const Product& q = p[i];
        for (int t = 0; t < (TAIL == GLU ? 2 : q.terms); t++) {
            if (t == 0 || TAIL != GLU) FH_TRY(map_of(&j.a[t], q.a[t], q.mn_a ? 64 : 128, dtype));
            FH_TRY(map_of(&j.b[t], q.b[t], q.mn_b || TAIL == GLU_AGAIN ? 64 : TAIL == GLU ? s.bn / 2 : nb, dtype));
        }
        const int kb = (int)((q.k + 63) / 64);
        j.mn_a = q.mn_a, j.mn_b = q.mn_b, j.kb[0] = kb, j.kb[1] = TAIL == GLU_AGAIN ? (q.a[1].cols + 63) / 64 : q.terms > 1 ? kb : 0, j.m = (int)q.m, j.n = q.n;
        j.tiles_m = (int)((q.m + 128 * s.ctas - 1) / (128 * s.ctas));
        const int cols = TAIL == GLU ? s.bn / 2 : TAIL == GLU_AGAIN ? kAgain : s.bn;
        j.tiles_n = (q.n + cols - 1) / cols;
        j.splits = s.splits[i];
        j.first = w.items;
        if ((long long)j.tiles_m * j.tiles_n > (1ll << 30) || (long long)j.tiles_n * kGroupM > (1ll << 30)) return cudaErrorInvalidValue;
        j.by_tiles = Divider((unsigned)(j.tiles_m * j.tiles_n)), j.by_group = Divider((unsigned)(kGroupM * j.tiles_n));
        const long long items = w.items + (long long)j.tiles_m * j.tiles_n * j.splits;
        if (items > (1ll << 30)) return cudaErrorInvalidValue;
        w.items = (int)items;
        j.out = q.out, j.pitch = q.pitch, j.bias0 = q.bias0, j.bias1 = q.bias1;
        w.out[0] = q.out1, w.out[1] = q.out2;
        auto tail_map = [&](CUtensorMap* map, const void* x, bool f32 = false) {
            return map_of(map, {x, q.pitch, q.m, q.n}, 0, f32 ? kF32 : dtype);
        };
        if (TAIL == GLU && q.out1) {
            w.keep = 1;
            FH_TRY(tail_map(&w.x[0], q.out1, true));
            FH_TRY(tail_map(&w.x[1], q.out2, true));
        }
        if (TAIL == GLU_AGAIN) {
            FH_TRY(tail_map(&w.x[0], q.out1));
            FH_TRY(tail_map(&w.x[1], q.out2));
            FH_TRY(map_of(&w.x[2], q.up, 64, dtype));
        }
        if (TAIL == GLU_GRAD) {
            FH_TRY(tail_map(&w.x[0], q.out1));
            FH_TRY(tail_map(&w.x[1], q.g, true));
            FH_TRY(tail_map(&w.x[2], q.u, true));
        }
        j.part = j.sums_part = nullptr;
        j.sums = q.sums;
        if (q.sums) w.sums = 1;
        if (j.splits > 1) {
            j.part = part;
            sums->s[sums->n++] = {part, q.out, q.bias0, q.pitch, q.m, q.n, j.splits, sums->total};
            sums->total += q.m * (((q.n + 7) & ~7) / 4);
            if (q.sums) {
                j.sums_part = part + product_part_floats(q, j.splits);
                sums->s[sums->n++] = {j.sums_part, q.sums, nullptr, q.m, 1, (int)q.m, j.splits, sums->total};
                sums->total += ((q.m + 7) & ~7) / 4;
            }
            part += part_floats(q, j.splits);
        } else {
            FH_TRY(tail_map(&j.o, q.out));
        }
    }
    if constexpr (TAIL != GLU_AGAIN)
        if (s.ctas == 2) return launch_work<T, 2, TAIL>(w, st);
    return launch_work<T, 1, TAIL>(w, st);
}
template <typename T>
cudaError_t finish(const Sums& sums, cudaStream_t st) {
    if (!sums.n) return cudaSuccess;
    return fhk::launch(k_sums<T>, dim3((unsigned)((sums.total + 31) / 32)), dim3(256), 0, st, sums);
}

// Whether a forward call takes the form for few rows: by estimates in us of both. It reads the weights at about 5.5 TB/s,
// slowed as every CTA reads 8 NT rows of x beside its 16 weight rows, with about 4 us of launches and latencies; the tiles
// need about 10 us and 5.2 TB/s whatever the rows. Measured (bf16, us, this form / tiles): 1 row of 1024 -> 4096 7.2 / 19,
// 32 rows 13.6 / 18.5; 2048 -> 8192 24 / 30 with 1 row, 32 / 30 with 16, 41 / 30 with 32; 4096 -> 16384 75 / 84 with 1, 109 / 84
// with 16.
bool takes_few_rows(long long m, int cin, int hidden, int cout) {
    if (m > 32) return false;
    const double mb = 2e-6 * hidden * (2.0 * cin + cout);
    const int nt = m <= 8 ? 1 : m <= 16 ? 2 : 4;
    return 4 + mb / 5.5 * (0.8 + 0.325 * nt) < 10 + mb / 5.2;
}
template <typename T, int NT, bool GATED>
cudaError_t launch_rows(const RowsArgs<T>& p, cudaStream_t st) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)((p.n + 15) / 16 * p.share));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    unsigned na = 0;
    if (p.share > 1) {
        at[na].id = cudaLaunchAttributeClusterDimension;
        at[na].val.clusterDim = {(unsigned)p.share, 1, 1};
        na++;
    }
    if (fhk::pdl_flag()) {
        at[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[na].val.programmaticStreamSerializationAllowed = 1;
        na++;
    }
    cfg.attrs = at;
    cfg.numAttrs = na;
    return cudaLaunchKernelEx(&cfg, k_rows<T, NT, GATED>, p);
}
template <typename T, bool GATED>
cudaError_t few_rows(const Product& q, int act, cudaStream_t st) {
    RowsArgs<T> p{};
    p.x = static_cast<const T*>(q.a[0].p), p.x_pitch = q.a[0].pitch;
    p.w0 = static_cast<const T*>(q.b[0].p), p.w0_pitch = q.b[0].pitch;
    if (GATED) p.w1 = static_cast<const T*>(q.b[1].p), p.w1_pitch = q.b[1].pitch;
    p.bias0 = static_cast<const T*>(q.bias0), p.bias1 = static_cast<const T*>(q.bias1);
    p.out = static_cast<T*>(q.out), p.g = static_cast<float*>(q.out1), p.u = static_cast<float*>(q.out2), p.pitch = q.pitch;
    p.m = (int)q.m, p.n = q.n, p.k = (int)q.k, p.act = act, p.share = 1;
    // a cluster per 16 channels until there is a CTA for every SM, while each warp keeps two steps of K
    while (p.share < 8 && (p.n + 15) / 16 * p.share < kSms && (p.k + 31) / 32 >= 32 * p.share) p.share *= 2;
    if (p.m <= 8) return launch_rows<T, 1, GATED>(p, st);
    if (p.m <= 16) return launch_rows<T, 2, GATED>(p, st);
    return launch_rows<T, 4, GATED>(p, st);
}

template <typename P>
bool good_sizes(const P* p) {
    return p->m >= 0 && p->m <= kMaxRows && p->cin >= 1 && p->cin <= kMaxChannels && p->hidden >= 1 &&
           p->hidden <= kMaxChannels && p->cout >= 1 && p->cout <= kMaxChannels && p->act >= FH_ACT_SILU &&
           p->act <= FH_ACT_SIGMOID && (p->dtype == FH_F16 || p->dtype == FH_BF16) && p->wait_cycles >= 0 &&
           p->test_extra_tx >= 0 && p->test_extra_tx <= 65536 && p->test_extra_tx % 16 == 0;
}
template <typename P>
bool good_weights(const P* p) {
    return good_rows(p->w_gate, p->wg_pitch, p->cin, p->hidden) && good_rows(p->w_up, p->wu_pitch, p->cin, p->hidden) &&
           good_rows(p->w_down, p->wd_pitch, p->hidden, p->cout);
}


// where the activated products go: the caller's a, else the scratch's first bytes
size_t own_a_bytes(const FhGatedFfnParams& p) { return p.a ? 0 : ((size_t)p.m * p.h_pitch * 2 + 255) / 256 * 256; }
void* a_of(const FhGatedFfnParams& p) { return p.a ? p.a : p.scratch; }
Product glu_of(const FhGatedFfnParams& p) {
    Product q{};
    q.a[0] = {p.x, p.x_pitch, p.m, p.cin};
    q.b[0] = {p.w_gate, p.wg_pitch, p.hidden, p.cin};
    q.b[1] = {p.w_up, p.wu_pitch, p.hidden, p.cin};
    q.terms = 1, q.m = p.m, q.n = p.hidden, q.k = p.cin;
    q.out = a_of(p), q.out1 = p.g, q.out2 = p.u, q.pitch = p.h_pitch, q.bias0 = p.b_gate, q.bias1 = p.b_up;
    return q;
}
Product down_of(const FhGatedFfnParams& p) {
    Product q{};
    q.a[0] = {a_of(p), p.h_pitch, p.m, p.hidden};
    q.b[0] = {p.w_down, p.wd_pitch, p.cout, p.hidden};
    q.terms = 1, q.m = p.m, q.n = p.cout, q.k = p.hidden, q.can_split = true;
    q.out = p.y, q.pitch = p.y_pitch, q.bias0 = p.b_down;
    return q;
}

// Whether a forward call runs as one kernel (gated_ffn_map.cuh): few channels, and nothing of the hidden values is kept (a alone
// is kept too: without g and u it cannot serve the gradient, but the caller reads it). It needs no scratch, and is the faster
// where tiles fill the SMs or hidden channels are few (f16, us, this form / tiles: 129,600 x 64 -> 256 32 / 49, 19,000 x 128 ->
// 16,384 434 / 468, 6480 x 48 -> 192 8.7 / 11.6); few tiles of many hidden channels go through few SMs one chunk after another
// and are slower by far (1000 x 128 -> 512 16 / 10, 8000 x 128 -> 4096 88 / 58, 64 x 128 -> 16,384 408 / 19).
bool on_map(const FhGatedFfnParams& p) { return !p.a && !p.g && p.cin <= kMapChannels && p.cout <= kMapChannels; }

template <typename T>
cudaError_t forward(const FhGatedFfnParams& p, cudaStream_t st) {
    const Product glu = glu_of(p), down = down_of(p);
    Sums sums{};
    if (takes_few_rows(p.m, p.cin, p.hidden, p.cout)) {
        FH_TRY((few_rows<T, true>(glu, p.act, st)));
        fhk::PdlScope pdl(true);
        return few_rows<T, false>(down, p.act, st);
    }
    if (on_map(p)) return block_on_map<T>(p, st);
    FH_TRY((products<T, GLU>(shape_of<GLU>(&glu, 1), &glu, 1, p, nullptr, nullptr, st)));
    fhk::PdlScope pdl(true);  // what follows waits on a kernel of this file
    FH_TRY((products<T, PLAIN>(shape_of<PLAIN>(&down, 1), &down, 1, p,
                                reinterpret_cast<float*>(static_cast<char*>(p.scratch) + own_a_bytes(p)), &sums, st)));
    return finish<T>(sums, st);
}

// the gradient's scratch: dg and du (and a, where it is formed again) [m][h_pitch], then the split sums and the partial
// column sums
struct GradPlan {
    Product da, out[kJobs];
    int outs;
    Shape shape;  // of out
    bool again;
    size_t hidden_bytes, all_hidden_bytes, part_bytes, column_bytes;
    ColumnSums cols;
    void* db[3];
    int ncols, widest;
};
GradPlan grad_plan(const FhGatedFfnGradParams& p) {
    GradPlan g{};
    g.hidden_bytes = ((size_t)p.m * p.h_pitch * 2 + 255) / 256 * 256;
    char* dg = static_cast<char*>(p.scratch);
    char* du = dg + g.hidden_bytes;
    g.again = !p.g;
    g.all_hidden_bytes = (g.again ? 3 : 2) * g.hidden_bytes;
    const void* a = g.again ? du + g.hidden_bytes : p.a;
    g.da.a[0] = {p.dy, p.dy_pitch, p.m, p.cout};
    g.da.b[0] = {p.w_down, p.wd_pitch, p.cout, p.hidden};
    g.da.mn_b = true;
    g.da.terms = 1, g.da.m = p.m, g.da.n = p.hidden, g.da.k = p.cout;
    g.da.out = dg, g.da.out1 = du, g.da.pitch = p.h_pitch, g.da.g = p.g, g.da.u = p.u;
    if (g.again) {
        g.da.terms = 2;
        g.da.a[1] = {p.x, p.x_pitch, p.m, p.cin};
        g.da.b[1] = {p.w_gate, p.wg_pitch, p.hidden, p.cin};
        g.da.up = {p.w_up, p.wu_pitch, p.hidden, p.cin};
        g.da.out2 = const_cast<void*>(a);
        g.da.bias0 = p.b_gate, g.da.bias1 = p.b_up;
    }
    if (p.dx) {
        Product& q = g.out[g.outs++];
        q.a[0] = {dg, p.h_pitch, p.m, p.hidden};
        q.a[1] = {du, p.h_pitch, p.m, p.hidden};
        q.b[0] = {p.w_gate, p.wg_pitch, p.hidden, p.cin};
        q.b[1] = {p.w_up, p.wu_pitch, p.hidden, p.cin};
        q.mn_b = true;
        q.terms = 2, q.m = p.m, q.n = p.cin, q.k = p.hidden, q.can_split = true, q.out = p.dx, q.pitch = p.dx_pitch;
    }
    Product* weights[3] = {};
    int which = 0;
    auto weight = [&](Matrix left, Matrix right, void* out, long long pitch) {
        which++;
        if (!out) return;
        Product& q = *(weights[which - 1] = &g.out[g.outs++]);
        q.a[0] = left, q.b[0] = right, q.mn_a = q.mn_b = true;
        q.terms = 1, q.m = left.cols, q.n = right.cols, q.k = p.m, q.can_split = true, q.out = out, q.pitch = pitch;
    };
    const Matrix x = {p.x, p.x_pitch, p.m, p.cin};
    weight({dg, p.h_pitch, p.m, p.hidden}, x, p.dw_gate, p.dwg_pitch);
    weight({du, p.h_pitch, p.m, p.hidden}, x, p.dw_up, p.dwu_pitch);
    weight({p.dy, p.dy_pitch, p.m, p.cout}, {a, p.h_pitch, p.m, p.hidden}, p.dw_down, p.dwd_pitch);
    // a bias's gradient is the row sums of its weight's gradient's left operand: taken along where the tiles leave tensor
    // memory for it, else by a pass of its own
    void* const db[3] = {p.db_gate, p.db_up, p.db_down};
    if (g.outs) g.shape = shape_of<PLAIN>(g.out, g.outs);
    const bool along = g.outs && g.shape.bn <= 128;
    for (int i = 0; i < 3; i++)
        if (along && weights[i]) weights[i]->sums = db[i];
    g.part_bytes = (g.outs ? scratch_floats(g.shape, g.out, g.outs) * 4 + 255 : 0) / 256 * 256;
    auto column = [&](const void* x_, long long pitch, int n, void* out) {
        if (!out) return;
        g.db[g.ncols] = out;
        g.cols.c[g.ncols++] = {x_, pitch, n, nullptr};
        g.widest = std::max(g.widest, n);
    };
    if (!along || !weights[0]) column(dg, p.h_pitch, p.hidden, p.db_gate);
    if (!along || !weights[1]) column(du, p.h_pitch, p.hidden, p.db_up);
    if (!along || !weights[2]) column(p.dy, p.dy_pitch, p.cout, p.db_down);
    if (g.ncols) {
        // about four CTAs per SM over the columns, 64 rows to a slice at least
        const long long across = (long long)((g.widest + 63) / 64) * g.ncols;
        g.cols.slices = (int)std::max<long long>(1, std::min<long long>((p.m + 63) / 64, 4 * kSms / across));
        g.cols.m = p.m;
        float* at = reinterpret_cast<float*>(dg + g.all_hidden_bytes + g.part_bytes);
        for (int i = 0; i < g.ncols; i++) {
            g.cols.c[i].part = at + g.column_bytes / 4;
            g.column_bytes += (size_t)g.cols.slices * ((g.cols.c[i].n + 7) & ~7) * 4;
        }
    }
    return g;
}

template <typename T>
cudaError_t gradient(const FhGatedFfnGradParams& p, const GradPlan& g, cudaStream_t st) {
    // whether dg or du is read (or a, formed with them)
    const bool hidden = p.dx || p.dw_gate || p.dw_up || p.db_gate || p.db_up || (g.again && p.dw_down);
    Sums sums{};
    if (hidden && g.again) FH_TRY((products<T, GLU_AGAIN>(shape_of<GLU_AGAIN>(&g.da, 1), &g.da, 1, p, nullptr, nullptr, st)));
    if (hidden && !g.again) FH_TRY((products<T, GLU_GRAD>(shape_of<GLU_GRAD>(&g.da, 1), &g.da, 1, p, nullptr, nullptr, st)));
    bool mine = hidden;  // whether the stream's last kernel is one of this file's, which the next may wait for itself
    if (g.outs) {
        fhk::PdlScope pdl(mine);
        FH_TRY((products<T, PLAIN>(g.shape, g.out, g.outs, p,
                                   reinterpret_cast<float*>(static_cast<char*>(p.scratch) + g.all_hidden_bytes), &sums, st)));
        mine = true;
    }
    if (g.ncols) {
        fhk::PdlScope pdl(mine);
        FH_TRY(fhk::launch(k_column_parts<T>, dim3((g.widest + 63) / 64, g.cols.slices, g.ncols), dim3(256), 0, st, g.cols));
        for (int i = 0; i < g.ncols; i++) {
            const Columns& c = g.cols.c[i];
            sums.s[sums.n++] = {c.part, g.db[i], nullptr, c.n, 1, c.n, g.cols.slices, sums.total};
            sums.total += ((c.n + 7) & ~7) / 4;
        }
        mine = true;
    }
    fhk::PdlScope pdl(mine);
    return finish<T>(sums, st);
}

}  // namespace

extern "C" size_t fhk_gated_ffn_scratch_bytes(const FhGatedFfnParams* p) {
    if (!p || !good_sizes(p) || p->m == 0 || p->h_pitch <= 0 || p->h_pitch > (1ll << 24)) return 0;
    if (takes_few_rows(p->m, p->cin, p->hidden, p->cout)) return own_a_bytes(*p);
    if (on_map(*p)) return 0;
    const Product down = down_of(*p);
    return own_a_bytes(*p) + scratch_floats(shape_of<PLAIN>(&down, 1), &down, 1) * 4;
}

extern "C" int fhk_gated_ffn(const FhGatedFfnParams* p, void* stream) {
    if (!p || !good_sizes(p) || !good_weights(p)) return (int)cudaErrorInvalidValue;
    if (!aligned16(p->b_gate) || !aligned16(p->b_up) || !aligned16(p->b_down)) return (int)cudaErrorInvalidValue;
    if (!good_rows(p->x, p->x_pitch, p->cin, p->m) || !good_rows(p->y, p->y_pitch, p->cout, p->m) ||
        !good_rows_or_null(p->a, p->h_pitch, p->hidden, p->m) || (p->g != nullptr) != (p->u != nullptr) || (p->g && !p->a) ||
        p->h_pitch < p->hidden || (p->h_pitch & 7) || p->h_pitch > (1ll << 24) ||
        !good_rows_or_null(p->g, p->h_pitch, p->hidden, p->m) || !good_rows_or_null(p->u, p->h_pitch, p->hidden, p->m))
        return (int)cudaErrorInvalidValue;
    const size_t need = fhk_gated_ffn_scratch_bytes(p);
    if (need && (!p->scratch || !aligned16(p->scratch) || p->scratch_bytes < need)) return (int)cudaErrorInvalidValue;
    if (p->m == 0) return 0;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return (int)(p->dtype == FH_F16 ? forward<__half>(*p, st) : forward<__nv_bfloat16>(*p, st));
}

extern "C" size_t fhk_gated_ffn_grad_scratch_bytes(const FhGatedFfnGradParams* p) {
    if (!p || !good_sizes(p) || p->m == 0 || p->h_pitch <= 0 || p->h_pitch > (1ll << 24)) return 0;
    const GradPlan g = grad_plan(*p);
    return g.all_hidden_bytes + g.part_bytes + g.column_bytes;
}

extern "C" int fhk_gated_ffn_grad(const FhGatedFfnGradParams* p, void* stream) {
    if (!p || !good_sizes(p) || !good_weights(p)) return (int)cudaErrorInvalidValue;
    if (!good_rows(p->x, p->x_pitch, p->cin, p->m) || !good_rows(p->dy, p->dy_pitch, p->cout, p->m) ||
        !good_rows_or_null(p->g, p->h_pitch, p->hidden, p->m) || !good_rows_or_null(p->u, p->h_pitch, p->hidden, p->m) ||
        !good_rows_or_null(p->a, p->h_pitch, p->hidden, p->m) || (p->g != nullptr) != (p->u != nullptr) ||
        (p->g != nullptr) != (p->a != nullptr) || p->h_pitch < p->hidden || (p->h_pitch & 7) || p->h_pitch > (1ll << 24) ||
        !good_rows_or_null(p->dx, p->dx_pitch, p->cin, p->m) ||
        !good_rows_or_null(p->dw_gate, p->dwg_pitch, p->cin, p->hidden) ||
        !good_rows_or_null(p->dw_up, p->dwu_pitch, p->cin, p->hidden) ||
        !good_rows_or_null(p->dw_down, p->dwd_pitch, p->hidden, p->cout))
        return (int)cudaErrorInvalidValue;
    if (!aligned16(p->db_gate) || !aligned16(p->db_up) || !aligned16(p->db_down) || !aligned16(p->b_gate) || !aligned16(p->b_up))
        return (int)cudaErrorInvalidValue;
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
    const GradPlan g = grad_plan(*p);
    if (!p->scratch || !aligned16(p->scratch) || p->scratch_bytes < g.all_hidden_bytes + g.part_bytes + g.column_bytes)
        return (int)cudaErrorInvalidValue;
    return (int)(p->dtype == FH_F16 ? gradient<__half>(*p, g, st) : gradient<__nv_bfloat16>(*p, g, st));
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
