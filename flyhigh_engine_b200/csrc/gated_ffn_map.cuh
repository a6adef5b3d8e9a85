// The whole block in one kernel for feature maps: up to 128 channels in and out, any hidden width, many rows.
//
// With few channels the hidden values are most of what a two-launch form would write and read back (2 F of 2 (F + C)
// elements a row), and its tiles have one or two K blocks each, so that what a tile costs besides its products decides.
// Here a CTA takes 128 rows (or two such tiles side by side) through the whole block: for each chunk of 64 hidden
// channels the gate and up projections land in one 128-column accumulator, the warps turn them into 64 columns of a, which
// go to shared memory as the A operand of the chunk's share of the down projection, and that accumulates in tensor memory
// over all chunks. The hidden values never leave the SM. The weights stay in shared memory where all chunks fit, else
// they pass through a ring (from L2).
//
// The biases of the projections enter as one more K step: a tile of ones' first column times a tile that holds the chunk's
// 128 biases in its first column, exact in the f32 accumulators, so that the activations' warps do not touch them (adding
// them there cost 8 of 39 us at 129,600 rows of 64 -> 256 -> 64).
//
// At that size the kernel takes 32 us, where the products alone would take 8. Nothing is full (special functions 41 %, issue
// slots 45 %, matrix pipe 20 %): what bounds it is the chain from accumulator to activation to operand, of which a group has
// one under way at a time. 6480 rows of 48 -> 192 -> 48, in 51 CTAs: 8.7 us.
#pragma once
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "ffn_parts.cuh"
#include "launch.h"

namespace {

constexpr int kMapChannels = 128, kMapChunk = 64;
constexpr int kMapEpi = 16, kMapThreads = (kMapEpi + 3) * 32;
// shared memory: x tiles, a's tiles (between items the staging tiles of the output), the weights' slots, the biases' tiles
constexpr int kMapX = 65536, kMapA = 32768, kMapW = 98304, kMapSlots = 4, kMapBias = 4096;
constexpr int kMapSmem = 1024 + kMapX + kMapA + kMapW + (1 + kMapSlots) * kMapBias + 256;
static_assert(kMapEpi * kTile == kMapA, "a staging tile per warp in a's place");

struct alignas(64) MapWork {
    CUtensorMap x, wg, wu, wd, y;
    int m, hidden, cout;
    int kb, ksteps;  // K blocks of 64 and steps of 16 of the projections
    int np;          // output columns rounded up to 32
    int chunks, slots, resident;
    int groups;      // 128-row tiles of a CTA, 1 or 2
    int tiles, act;
    int extra;       // bytes that x's barrier expects beyond its copies (0, or a test's)
    const void *b_gate, *b_up, *b_down;
    void* out;
    long long pitch, limit;
};

template <typename T>
__global__ void __launch_bounds__(kMapThreads, 1) k_block(const __grid_constant__ MapWork w) {
    extern __shared__ uint8_t raw[];
    using namespace umma;
    const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
    const uint32_t xs = base, as = xs + kMapX, ws = as + kMapA, ones = ws + kMapW, bias = ones + kMapBias, bars = bias + kMapSlots * kMapBias;
    const uint32_t xfull = bars, xempty = bars + 16, wfull = bars + 32, wempty = bars + 64, d1full = bars + 96, d1empty = bars + 112,
                   afull = bars + 128, aempty = bars + 144, d2full = bars + 160, d2empty = bars + 176, stored = bars + 192, slot_at = bars + 208;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int kb = w.kb, chunks = w.chunks, groups = w.groups, xbufs = kb == 1 ? 2 : 1;
    const uint32_t xtile = kb * 16384, wbytes = kb * 16384 + w.np * 128;
    const bool bf16 = !std::is_same<T, __half>::value, biased = w.b_gate || w.b_up;

    if (warp == 16 && lane == 0) {
        for (int i = 0; i < 2; i++) {
            bar_init(xfull + 8 * i, 1), bar_init(xempty + 8 * i, groups);
            bar_init(d1full + 8 * i, 1), bar_init(d1empty + 8 * i, 8);
            bar_init(afull + 8 * i, 8), bar_init(aempty + 8 * i, 1);
            bar_init(d2full + 8 * i, 1), bar_init(d2empty + 8 * i, 8), bar_init(stored + 8 * i, 8);
        }
        for (int i = 0; i < kMapSlots; i++) bar_init(wfull + 8 * i, biased ? 2 : 1), bar_init(wempty + 8 * i, groups);
        bar_init_fence();
    }
    if (biased) {  // the tile of ones, and zeros under the biases
        for (int i = threadIdx.x; i < (1 + kMapSlots) * kMapBias / 4; i += kMapThreads) {
            const bool one = i < kMapBias / 4 && (i & 63) < 32 && (i & 3) == 0;  // first word of a row's first half
            asm volatile("st.shared.b32 [%0], %1;\n" ::"r"(ones + 4 * i), "r"(one ? (bf16 ? 0x3f80u : 0x3c00u) : 0u) : "memory");
        }
        fence_async();
    }
    if (warp == 17) tmem_alloc<1>(slot_at, 512);
    fence_before();
    __syncthreads();
    fence_after();
    uint32_t tbase;
    asm volatile("ld.shared.b32 %0, [%1];\n" : "=r"(tbase) : "r"(slot_at));
    tbase = uniform(tbase);
    pdl_wait();
    pdl_trigger();

    bool ok = true;
    auto wait = [&](uint32_t bar, uint32_t parity) {  // by whole warps
        if (ok) ok = __all_sync(0xffffffffu, bar_wait(bar, parity & 1, w.limit, &g_ffn_timeouts));
        return ok;
    };
    // group g takes tiles blockIdx.x + gridDim.x (groups n + g), so that the last tiles go to different CTAs
    auto tile_of = [&](int n, int g) { return (int)blockIdx.x + (int)gridDim.x * (groups * n + g); };
    if (warp == 16) {
        const bool leader = elected();
        int s = 0;
        uint32_t ph = 1;  // the ring starts empty
        for (int n = 0; ok && tile_of(n, 0) < w.tiles; n++) {
            const int b = n % xbufs;
            if (!wait(xempty + 8 * b, n / xbufs + 1)) break;
            if (leader) {
                const int live = groups == 2 && tile_of(n, 1) < w.tiles ? 2 : 1;
                bar_expect(xfull + 8 * b, live * xtile + w.extra);
                for (int g = 0; g < live; g++)
                    for (int k = 0; k < kb; k++)
                        tensor_load<1>(xs + (b * 2 + g) * xtile + k * 16384, &w.x, k * BK, tile_of(n, g) * 128, xfull + 8 * b);
            }
            __syncwarp();
            if (w.resident && n > 0) continue;
            for (int c = 0; c < chunks; c++) {
                if (!wait(wempty + 8 * s, ph)) break;
                const uint32_t at = ws + s * wbytes, bar = wfull + 8 * s;
                if (leader) {
                    bar_expect(bar, wbytes);
                    for (int k = 0; k < kb; k++) {
                        tensor_load<1>(at + k * 16384, &w.wg, k * BK, c * kMapChunk, bar);
                        tensor_load<1>(at + k * 16384 + 8192, &w.wu, k * BK, c * kMapChunk, bar);
                    }
                    tensor_load<1>(at + kb * 16384, &w.wd, c * kMapChunk, 0, bar);
                }
                __syncwarp();
                if (biased) {  // row r of the bias tile (gate 0-63, up 64-127): 8-row group r / 8, 16 bytes a row
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int r = lane + 32 * e, col = c * kMapChunk + (r & 63);
                        const T* v = static_cast<const T*>(e < 2 ? w.b_gate : w.b_up);
                        const T val = v && col < w.hidden ? v[col] : Elem<T>::from(0.0f);
                        asm volatile("st.shared.b16 [%0], %1;\n" ::"r"(bias + s * kMapBias + (r >> 3) * 256 + (r & 7) * 16),
                                     "h"(*reinterpret_cast<const unsigned short*>(&val))
                                     : "memory");
                    }
                    fence_async();
                    __syncwarp();
                    if (lane == 0) bar_arrive(bar);
                }
                if (++s == w.slots) s = 0, ph ^= 1;
            }
        }
    } else if (warp >= 17) {
        // one issuing warp per tile: an issuer takes about 60 cycles for a matrix instruction and more for a commit, and the
        // two tiles go at their own pace
        const int g = warp - 17;
        const uint32_t id1 = instr_desc(bf16, false, false, 128, 128), id2 = instr_desc(bf16, false, false, 128, w.np);
        const uint32_t d1 = tbase + g * 128, d2 = tbase + 256 + g * 128;
        const uint64_t a2 = tile_desc(as + g * 16384, 0);
        const bool leader = elected();
        int u = 0, s = 0;  // u: chunks so far; s: the ring's slot of the next chunk
        uint32_t ph = 0;
        for (int n = 0; g < groups && ok && tile_of(n, 0) < w.tiles; n++) {
            const int b = n % xbufs;
            if (tile_of(n, g) >= w.tiles) {  // only the other group has a last tile: let its weights pass
                for (int c = 0; c < chunks && !w.resident; c++) {
                    if (!wait(wfull + 8 * s, ph)) break;
                    if (leader) bar_arrive(wempty + 8 * s);
                    if (++s == w.slots) s = 0, ph ^= 1;
                }
                break;
            }
            if (!wait(xfull + 8 * b, n / xbufs)) break;
            int last = 0;  // the slot of the chunk before
            for (int c = 0; c <= chunks; c++) {
                const int here = w.resident ? c : s;
                if (c < chunks) {
                    if ((!w.resident || n == 0) && !wait(wfull + 8 * here, ph)) break;
                    if (!wait(d1empty + 8 * g, u + 1)) break;
                    fence_after();
                    const uint64_t ad = tile_desc(xs + (b * 2 + g) * xtile, 0), bd = tile_desc(ws + here * wbytes, 0);
                    if (leader) {
                        for (int k = 0; k < w.ksteps; k += 4) {
                            const uint32_t o = (k >> 2) * (16384 >> 4);
                            mma<1>(d1, ad + o, bd + o, id1, k > 0);
#pragma unroll
                            for (int e = 1; e < 4; e++)
                                if (k + e < w.ksteps) mma<1>(d1, ad + o + e * (32 >> 4), bd + o + e * (32 >> 4), id1, 1);
                        }
                        if (biased) mma<1>(d1, plain_desc(ones), plain_desc(bias + here * kMapBias), id1, 1);
                        commit<1>(d1full + 8 * g);
                        if (c == chunks - 1) commit<1>(xempty + 8 * b);
                    }
                }
                if (c > 0) {
                    if (!wait(afull + 8 * g, u - 1)) break;
                    if (c == 1 && !wait(d2empty + 8 * g, n + 1)) break;
                    fence_after();
                    const uint64_t bd = tile_desc(ws + last * wbytes + kb * 16384, 0);
                    if (leader) {
                        mma<1>(d2, a2, bd, id2, c > 1);
#pragma unroll
                        for (int k = 1; k < 4; k++) mma<1>(d2, a2 + k * (32 >> 4), bd + k * (32 >> 4), id2, 1);
                        commit<1>(aempty + 8 * g);
                        if (c == chunks) commit<1>(d2full + 8 * g);
                        if (!w.resident) commit<1>(wempty + 8 * last);
                    }
                }
                last = here;
                if (c < chunks) {
                    u++;
                    if (++s == w.slots) s = 0, ph ^= 1;
                }
            }
        }
    } else if (warp / 8 < groups) {
        const int g = warp >> 3, q = warp & 3, half = (warp >> 2) & 1, r = q * 32 + lane;
        const uint32_t acc1 = tbase + ((uint32_t)(q * 32) << 16) + g * 128 + half * 32, acc2 = tbase + ((uint32_t)(q * 32) << 16) + 256 + g * 128;
        const uint32_t arow = as + g * 16384 + r * 128, tile = as + warp * kTile;
        const bool ragged = w.cout & 7;
        const int span = w.np <= 64 ? 32 : 64, lo = half * span, hi = min(w.np, lo + span);
        uint32_t u = 0;
        for (int n = 0; tile_of(n, g) < w.tiles; n++) {
            if (n > 0) {  // the group's last output has left a's place
                if (lane == 0) {
                    stores_read<0>();
                    bar_arrive(stored + 8 * g);
                }
                __syncwarp();
                if (!wait(stored + 8 * g, n - 1)) break;
            }
            for (int c = 0; c < chunks; c++, u++) {
                wait(d1full + 8 * g, u);
                if (!ok) break;
                fence_after();
                // all of the chunk's columns at once: the next chunk's projections run while these are worked on
                uint32_t rg[32], ru[32];
                load32(acc1, rg);
                load32(acc1 + 64, ru);
                wait_ld();
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(d1empty + 8 * g);
                __syncwarp();
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float2 v[8], gv[8], uv[8];
                    pairs(rg + 16 * h, gv);
                    pairs(ru + 16 * h, uv);
                    switch (w.act) {
                        case FH_ACT_SILU: glu16<FH_ACT_SILU>(gv, uv, v); break;
                        case FH_ACT_GELU: glu16<FH_ACT_GELU>(gv, uv, v); break;
                        case FH_ACT_GELU_TANH: glu16<FH_ACT_GELU_TANH>(gv, uv, v); break;
                        case FH_ACT_RELU: glu16<FH_ACT_RELU>(gv, uv, v); break;
                        default: glu16<FH_ACT_SIGMOID>(gv, uv, v); break;
                    }
                    if (h == 0) {  // the down projection of the chunk before has read a's place
                        wait(aempty + 8 * g, u + 1);
                        if (!ok) break;
                    }
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(arow + (((4 * half + 2 * h + e) ^ (r & 7)) << 4)),
                                     "r"(Elem<T>::from2(v[4 * e].x, v[4 * e].y)), "r"(Elem<T>::from2(v[4 * e + 1].x, v[4 * e + 1].y)),
                                     "r"(Elem<T>::from2(v[4 * e + 2].x, v[4 * e + 2].y)), "r"(Elem<T>::from2(v[4 * e + 3].x, v[4 * e + 3].y))
                                     : "memory");
                    __syncwarp();
                }
                if (!ok) break;
                fence_async();
                __syncwarp();
                if (lane == 0) bar_arrive(afull + 8 * g);
            }
            if (!ok) break;
            wait(d2full + 8 * g, n);
            if (!ok) break;
            fence_after();
            const int row = tile_of(n, g) * 128 + q * 32;
            for (int c0 = lo; c0 < hi; c0 += 32) {
                if (lane == 0) stores_read<0>();
                __syncwarp();
                uint32_t r0[32];
                load32(acc2 + c0, r0);
                wait_ld();
                if (c0 + 32 >= hi) {
                    fence_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive(d2empty + 8 * g);
                }
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float2 v[8];
                    pairs(r0 + 16 * h, v);
                    if (w.b_down) {
                        uint32_t qb[8];
                        load_bias<T>(w.b_down, c0 + 16 * h, w.cout, qb);
                        add_bias<T>(qb, v);
                    }
                    tile_put<T>(tile, lane, h, v);
                }
                fence_async();
                __syncwarp();
                if (row < w.m && c0 < w.cout) {
                    if (ragged && c0 + 32 > w.cout) {  // the columns end inside a 16-byte piece
                        if (row + lane < w.m)
                            tile_out<T>(tile, lane, static_cast<T*>(w.out) + (long long)(row + lane) * w.pitch + c0, w.cout - c0);
                        __syncwarp();
                    } else if (lane == 0) {
                        tensor_store(&w.y, c0, row, tile);
                        stores_commit();
                    }
                }
            }
            if (lo >= hi) {
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(d2empty + 8 * g);
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
    __syncthreads();
    fence_after();
    if (warp == 17) tmem_free<1>(tbase, 512);
}

template <typename T>
cudaError_t block_on_map(const FhGatedFfnParams& p, cudaStream_t st) {
    static std::atomic<bool> prepared[64];  // per device
    int dev = 0;
    FH_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!prepared[dev].load(std::memory_order_acquire)) {
        FH_TRY(cudaFuncSetAttribute(k_block<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMapSmem));
        prepared[dev].store(true, std::memory_order_release);
    }
    MapWork w;
    w.m = (int)p.m, w.hidden = p.hidden, w.cout = p.cout, w.act = p.act, w.extra = p.test_extra_tx;
    w.kb = (p.cin + 63) / 64, w.ksteps = (p.cin + 15) / 16, w.np = (p.cout + 31) / 32 * 32;
    w.chunks = (p.hidden + kMapChunk - 1) / kMapChunk;
    w.slots = std::min(kMapSlots, kMapW / (w.kb * 16384 + w.np * 128));
    w.resident = w.chunks <= w.slots;
    // two tiles side by side (one's products run while the other's activations do) once every SM has one
    w.tiles = (int)((p.m + 127) / 128);
    w.groups = w.tiles > kSms ? 2 : 1;
    w.b_gate = p.b_gate, w.b_up = p.b_up, w.b_down = p.b_down;
    w.out = p.y, w.pitch = p.y_pitch, w.limit = p.wait_cycles > 0 ? p.wait_cycles : 2000000000ll;
    FH_TRY(map_of(&w.x, {p.x, p.x_pitch, p.m, p.cin}, 128, p.dtype));
    FH_TRY(map_of(&w.wg, {p.w_gate, p.wg_pitch, p.hidden, p.cin}, 64, p.dtype));
    FH_TRY(map_of(&w.wu, {p.w_up, p.wu_pitch, p.hidden, p.cin}, 64, p.dtype));
    FH_TRY(map_of(&w.wd, {p.w_down, p.wd_pitch, p.cout, p.hidden}, w.np, p.dtype));
    FH_TRY(map_of(&w.y, {p.y, p.y_pitch, p.m, p.cout}, 0, p.dtype));
    return fhk::launch(k_block<T>, dim3((unsigned)std::min(w.tiles, kSms)), dim3(kMapThreads), kMapSmem, st, w);
}

}  // namespace
