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
// Bound by the special functions: two a hidden value (exp, reciprocal), 16 per cycle and SM.
#pragma once
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "ffn_parts.cuh"
#include "launch.h"

namespace {

constexpr int kMapChannels = 128, kMapChunk = 64;
constexpr int kMapEpi = 16, kMapThreads = (kMapEpi + 2) * 32;
constexpr int kMapX = 65536, kMapA = 32768, kMapStage = kMapEpi * kTile, kMapW = 98304, kMapSlots = 4;
constexpr int kMapSmem = 1024 + kMapX + kMapA + kMapStage + kMapW + 256;

struct alignas(64) MapWork {
    CUtensorMap x, wg, wu, wd, y;
    int m, hidden, cout;
    int kb, ksteps;  // K blocks of 64 and steps of 16 of the projections
    int np;          // output columns rounded up to 32
    int chunks, slots, resident;
    int groups;      // 128-row tiles of a CTA, 1 or 2
    int items, act;
    const void *b_gate, *b_up, *b_down;
    void* out;
    long long pitch, limit;
};

template <typename T>
__global__ void __launch_bounds__(kMapThreads, 1) k_block(const __grid_constant__ MapWork w) {
    extern __shared__ uint8_t raw[];
    using namespace umma;
    const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
    const uint32_t xs = base, as = xs + kMapX, stage = as + kMapA, ws = stage + kMapStage, bars = ws + kMapW;
    const uint32_t xfull = bars, xempty = bars + 16, wfull = bars + 32, wempty = bars + 64, d1full = bars + 96, d1empty = bars + 112,
                   afull = bars + 128, aempty = bars + 144, d2full = bars + 160, d2empty = bars + 176, slot_at = bars + 192;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int kb = w.kb, chunks = w.chunks, groups = w.groups, xbufs = kb == 1 ? 2 : 1;
    const uint32_t xtile = kb * 16384, wbytes = kb * 16384 + w.np * 128;
    const bool bf16 = !std::is_same<T, __half>::value;

    if (warp == 16 && lane == 0) {
        for (int i = 0; i < 2; i++) {
            bar_init(xfull + 8 * i, 1), bar_init(xempty + 8 * i, 1);
            bar_init(d1full + 8 * i, 1), bar_init(d1empty + 8 * i, 8);
            bar_init(afull + 8 * i, 8), bar_init(aempty + 8 * i, 1);
            bar_init(d2full + 8 * i, 1), bar_init(d2empty + 8 * i, 8);
        }
        for (int i = 0; i < kMapSlots; i++) bar_init(wfull + 8 * i, 1), bar_init(wempty + 8 * i, 1);
        bar_init_fence();
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
    if (warp == 16) {
        int n = 0, wi = 0, s = 0;
        for (int i = blockIdx.x; ok && i < w.items; i += gridDim.x, n++) {
            const int b = n % xbufs;
            if (!wait(xempty + 8 * b, n / xbufs + 1)) break;
            if (lane == 0) {
                bar_expect(xfull + 8 * b, groups * xtile);
                for (int g = 0; g < groups; g++)
                    for (int k = 0; k < kb; k++)
                        tensor_load<1>(xs + (b * 2 + g) * xtile + k * 16384, &w.x, k * BK, (i * groups + g) * 128, xfull + 8 * b);
            }
            __syncwarp();
            if (w.resident && n > 0) continue;
            for (int c = 0; c < chunks; c++, wi++) {
                if (!wait(wempty + 8 * s, wi / w.slots + 1)) break;
                const uint32_t at = ws + s * wbytes, bar = wfull + 8 * s;
                if (lane == 0) {
                    bar_expect(bar, wbytes);
                    for (int k = 0; k < kb; k++) {
                        tensor_load<1>(at + k * 16384, &w.wg, k * BK, c * kMapChunk, bar);
                        tensor_load<1>(at + k * 16384 + 8192, &w.wu, k * BK, c * kMapChunk, bar);
                    }
                    tensor_load<1>(at + kb * 16384, &w.wd, c * kMapChunk, 0, bar);
                }
                __syncwarp();
                if (++s == w.slots) s = 0;
            }
        }
    } else if (warp == 17) {
        const uint32_t id1 = instr_desc(bf16, false, false, 128, 128), id2 = instr_desc(bf16, false, false, 128, w.np);
        int n = 0, u = 0, s = 0, wi = 0;  // u: chunks so far; s: the ring's slot of the next chunk
        for (int i = blockIdx.x; ok && i < w.items; i += gridDim.x, n++) {
            const int b = n % xbufs;
            if (!wait(xfull + 8 * b, n / xbufs)) break;
            int last = 0;  // the slot of the chunk before
            for (int c = 0; c <= chunks && ok; c++) {
                const int here = w.resident ? c : s;
                if (c < chunks) {
                    if ((!w.resident || n == 0) && !wait(wfull + 8 * here, wi / w.slots)) break;
                    for (int g = 0; g < groups; g++) {
                        if (!wait(d1empty + 8 * g, u + 1)) break;
                        fence_after();
                        uint64_t ad = tile_desc(xs + (b * 2 + g) * xtile, 0), bd = tile_desc(ws + here * wbytes, 0);
                        for (int k = 0; k < w.ksteps; k++) {
                            if (lane == 0) mma<1>(tbase + g * 128, ad, bd, id1, k > 0);
                            const uint32_t step = (k & 3) == 3 ? (16384 - 96) >> 4 : 32 >> 4;  // the next 16 of K, or K block
                            ad += step, bd += step;
                        }
                        if (lane == 0) commit<1>(d1full + 8 * g);
                    }
                    if (!ok) break;
                    if (c == chunks - 1 && lane == 0) commit<1>(xempty + 8 * b);
                }
                if (c > 0) {
                    for (int g = 0; g < groups; g++) {
                        if (!wait(afull + 8 * g, u - 1)) break;
                        if (c == 1 && !wait(d2empty + 8 * g, n + 1)) break;
                        fence_after();
                        const uint64_t ad = tile_desc(as + g * 16384, 0), bd = tile_desc(ws + last * wbytes + kb * 16384, 0);
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            if (lane == 0) mma<1>(tbase + 256 + g * 128, ad + k * (32 >> 4), bd + k * (32 >> 4), id2, c > 1 || k > 0);
                        if (lane == 0) {
                            commit<1>(aempty + 8 * g);
                            if (c == chunks) commit<1>(d2full + 8 * g);
                        }
                    }
                    if (!ok) break;
                    if (!w.resident && lane == 0) commit<1>(wempty + 8 * last);
                }
                last = here;
                if (c < chunks) {
                    u++, wi++;
                    if (++s == w.slots) s = 0;
                }
            }
        }
    } else if (warp / 8 < groups) {
        const int g = warp >> 3, q = warp & 3, half = (warp >> 2) & 1, r = q * 32 + lane;
        const uint32_t acc1 = tbase + ((uint32_t)(q * 32) << 16) + g * 128 + half * 32, acc2 = tbase + ((uint32_t)(q * 32) << 16) + 256 + g * 128;
        const uint32_t arow = as + g * 16384 + r * 128, tile = stage + warp * kTile;
        const bool biased = w.b_gate || w.b_up, ragged = w.cout & 7;
        const int span = w.np <= 64 ? 32 : 64, lo = half * span, hi = min(w.np, lo + span);
        int n = 0;
        uint32_t u = 0;
        for (int i = blockIdx.x; i < w.items; i += gridDim.x, n++) {
            for (int c = 0; c < chunks; c++, u++) {
                wait(d1full + 8 * g, u);
                if (!ok) break;
                fence_after();
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t rg[16], ru[16], qg[8], qu[8];
                    load16(acc1 + 16 * h, rg);
                    load16(acc1 + 64 + 16 * h, ru);
                    const int col = c * kMapChunk + half * 32 + 16 * h;
                    if (biased) {
                        load_bias<T>(w.b_gate, col, w.hidden, qg);
                        load_bias<T>(w.b_up, col, w.hidden, qu);
                        __syncwarp();
                    }
                    wait_ld();
                    if (h == 1) {
                        fence_before();
                        __syncwarp();
                        if (lane == 0) bar_arrive(d1empty + 8 * g);
                    }
                    float2 v[8], gv[8], uv[8];
                    pairs(rg, gv);
                    pairs(ru, uv);
                    if (biased) {
                        add_bias<T>(qg, gv);
                        add_bias<T>(qu, uv);
                    }
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
            const int row = (i * groups + g) * 128 + q * 32;
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
    w.m = (int)p.m, w.hidden = p.hidden, w.cout = p.cout, w.act = p.act;
    w.kb = (p.cin + 63) / 64, w.ksteps = (p.cin + 15) / 16, w.np = (p.cout + 31) / 32 * 32;
    w.chunks = (p.hidden + kMapChunk - 1) / kMapChunk;
    w.slots = std::min(kMapSlots, kMapW / (w.kb * 16384 + w.np * 128));
    w.resident = w.chunks <= w.slots;
    // two tiles side by side (one's products run while the other's activations do) once every SM has one
    const int tiles = (int)((p.m + 127) / 128);
    w.groups = tiles > kSms ? 2 : 1;
    w.items = (tiles + w.groups - 1) / w.groups;
    w.b_gate = p.b_gate, w.b_up = p.b_up, w.b_down = p.b_down;
    w.out = p.y, w.pitch = p.y_pitch, w.limit = p.wait_cycles > 0 ? p.wait_cycles : 2000000000ll;
    FH_TRY(map_of(&w.x, {p.x, p.x_pitch, p.m, p.cin}, 128, p.dtype));
    FH_TRY(map_of(&w.wg, {p.w_gate, p.wg_pitch, p.hidden, p.cin}, 64, p.dtype));
    FH_TRY(map_of(&w.wu, {p.w_up, p.wu_pitch, p.hidden, p.cin}, 64, p.dtype));
    FH_TRY(map_of(&w.wd, {p.w_down, p.wd_pitch, p.cout, p.hidden}, w.np, p.dtype));
    FH_TRY(map_of(&w.y, {p.y, p.y_pitch, p.m, p.cout}, 0, p.dtype));
    return fhk::launch(k_block<T>, dim3((unsigned)std::min(w.items, kSms)), dim3(kMapThreads), kMapSmem, st, w);
}

}  // namespace
