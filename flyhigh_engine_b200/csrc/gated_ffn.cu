// The gated feed-forward block (fhk_gated_ffn) and its gradient.
//
//   g = x Wg^T + bg, u = x Wu^T + bu, a = act(g) u, y = a Wd^T + bd
//   da = dy Wd; dg = da u act'(g), du = da act(g); dx = dg Wg + du Wu; dWg = dg^T x, dWu = du^T x, dWd = dy^T a
//
// Every one of these is a product over rows or channels with an elementwise tail. This is the plain form: one tiled
// kernel on the FMA units whose operands are addressed by two strides each, with the tails as template parameters.
#include <cuda_runtime.h>

#include <algorithm>

#include "fh_device.cuh"
#include "fh_kernels.h"
#include "launch.h"
#include "row_ops.cuh"

using namespace rows;

namespace {

constexpr int kMaxChannels = 1 << 20;

// act(g) and its derivative
__device__ __forceinline__ void act_both(int act, float g, float& v, float& dv) {
    if (act == FH_ACT_SILU || act == FH_ACT_SIGMOID) {
        const float s = 1.0f / (1.0f + __expf(-g));
        v = act == FH_ACT_SILU ? g * s : s;
        dv = act == FH_ACT_SILU ? s * (1.0f + g * (1.0f - s)) : s * (1.0f - s);
    } else if (act == FH_ACT_RELU) {
        v = g > 0.0f ? g : 0.0f;
        dv = g > 0.0f ? 1.0f : 0.0f;
    } else if (act == FH_ACT_GELU) {
        const float cdf = 0.5f * (1.0f + erff(g * 0.70710678f));
        v = g * cdf;
        dv = cdf + g * 0.39894228f * __expf(-0.5f * g * g);
    } else {
        const float k = 0.79788456f, t = tanhf(k * (g + 0.044715f * g * g * g));
        v = 0.5f * g * (1.0f + t);
        dv = 0.5f * (1.0f + t) + 0.5f * g * (1.0f - t * t) * k * (1.0f + 0.134145f * g * g);
    }
}

struct Operand {  // element (i, k) at p[i * si + k * sk]
    const void* p;
    long long si, sk;
};
enum Tail { PLAIN, GLU, GLU_GRAD };
struct Product {
    Operand a[2], b[2];  // PLAIN: sum of `terms` products; GLU: a[0] with b[0] and with b[1]
    long long m, n, k;
    int terms;
    void *out, *out1, *out2;  // PLAIN: out; GLU: a, and g, u or NULL; GLU_GRAD: dg, du
    long long pitch;
    const void *bias0, *bias1;  // by column
    const void *g, *u;          // GLU_GRAD
    int act;
};

template <typename T, int TAIL>
__global__ void __launch_bounds__(256) k_product(const Product q) {
    constexpr int NACC = TAIL == GLU ? 2 : 1;
    __shared__ float as[16][65], bs[NACC][16][65];
    const long long m0 = (long long)blockIdx.y * 64, n0 = (long long)blockIdx.x * 64;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float acc[NACC][4][4] = {};
    const int terms = TAIL == GLU ? 1 : q.terms;
    for (int t = 0; t < terms; t++)
        for (long long k0 = 0; k0 < q.k; k0 += 16) {
            for (int i = threadIdx.x; i < 1024; i += 256) {
                const int r = i / 16, kk = i % 16;
                as[kk][r] = m0 + r < q.m && k0 + kk < q.k
                                ? Elem<T>::to(static_cast<const T*>(q.a[t].p)[(m0 + r) * q.a[t].si + (k0 + kk) * q.a[t].sk])
                                : 0.0f;
                for (int w = 0; w < NACC; w++) {
                    const Operand& b = q.b[TAIL == GLU ? w : t];
                    bs[w][kk][r] = n0 + r < q.n && k0 + kk < q.k
                                       ? Elem<T>::to(static_cast<const T*>(b.p)[(n0 + r) * b.si + (k0 + kk) * b.sk])
                                       : 0.0f;
                }
            }
            __syncthreads();
            for (int kk = 0; kk < 16; kk++)
                for (int w = 0; w < NACC; w++)
                    for (int i = 0; i < 4; i++)
                        for (int j = 0; j < 4; j++) acc[w][i][j] += as[kk][ty + 16 * i] * bs[w][kk][tx + 16 * j];
            __syncthreads();
        }
    for (int i = 0; i < 4; i++)
        for (int j = 0; j < 4; j++) {
            const long long r = m0 + ty + 16 * i, c = n0 + tx + 16 * j;
            if (r >= q.m || c >= q.n) continue;
            const long long at = r * q.pitch + c;
            const float b0 = q.bias0 ? Elem<T>::to(static_cast<const T*>(q.bias0)[c]) : 0.0f;
            float v, dv;
            if (TAIL == PLAIN) {
                static_cast<T*>(q.out)[at] = Elem<T>::from(acc[0][i][j] + b0);
            } else if (TAIL == GLU) {
                const float b1 = q.bias1 ? Elem<T>::to(static_cast<const T*>(q.bias1)[c]) : 0.0f;
                const float g = acc[0][i][j] + b0, u = acc[NACC - 1][i][j] + b1;
                act_both(q.act, g, v, dv);
                static_cast<T*>(q.out)[at] = Elem<T>::from(v * u);
                if (q.out1) {
                    static_cast<T*>(q.out1)[at] = Elem<T>::from(g);
                    static_cast<T*>(q.out2)[at] = Elem<T>::from(u);
                }
            } else {
                act_both(q.act, Elem<T>::to(static_cast<const T*>(q.g)[at]), v, dv);
                const float u = Elem<T>::to(static_cast<const T*>(q.u)[at]);
                static_cast<T*>(q.out)[at] = Elem<T>::from(acc[0][i][j] * u * dv);
                static_cast<T*>(q.out1)[at] = Elem<T>::from(acc[0][i][j] * v);
            }
        }
}

// column sums of up to 64 rows x 32 columns per step, one CTA per 32 columns
template <typename T>
__global__ void __launch_bounds__(256) k_column_sums(const void* x, long long pitch, long long m, int n, void* out) {
    __shared__ float s[8][33];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), w = threadIdx.x >> 5;
    float v = 0.0f;
    if (c < n)
        for (long long r = w; r < m; r += 8) v += Elem<T>::to(static_cast<const T*>(x)[r * pitch + c]);
    s[w][threadIdx.x & 31] = v;
    __syncthreads();
    if (w == 0 && c < n) {
        v = 0.0f;
        for (int i = 0; i < 8; i++) v += s[i][threadIdx.x & 31];
        static_cast<T*>(out)[c] = Elem<T>::from(v);
    }
}

template <typename T, int TAIL>
cudaError_t product(const Product& q, cudaStream_t st) {
    // rows along gridDim.y (at most 65,535): in slices of rows for more
    for (long long m0 = 0; m0 < q.m; m0 += 65535ll * 64) {
        Product s = q;
        s.m = std::min<long long>(q.m - m0, 65535ll * 64);
        auto shift = [&](const void* p, long long by) -> void* {
            return p ? static_cast<char*>(const_cast<void*>(p)) + 2 * by : nullptr;
        };
        for (int t = 0; t < 2; t++) s.a[t].p = shift(q.a[t].p, m0 * q.a[t].si);
        s.out = shift(q.out, m0 * q.pitch);
        s.out1 = shift(q.out1, m0 * q.pitch);
        s.out2 = shift(q.out2, m0 * q.pitch);
        s.g = shift(q.g, m0 * q.pitch);
        s.u = shift(q.u, m0 * q.pitch);
        const cudaError_t e = fhk::launch(k_product<T, TAIL>, dim3((unsigned)((s.n + 63) / 64), (unsigned)((s.m + 63) / 64)),
                                          dim3(256), 0, st, s);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}
template <typename T>
cudaError_t column_sums(const void* x, long long pitch, long long m, int n, void* out, cudaStream_t st) {
    return fhk::launch(k_column_sums<T>, dim3((n + 31) / 32), dim3(256), 0, st, x, pitch, m, n, out);
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

#define FH_TRY(call)                              \
    do {                                          \
        const cudaError_t e_ = (call);            \
        if (e_ != cudaSuccess) return e_;         \
    } while (0)

template <typename T>
cudaError_t forward(const FhGatedFfnParams& p, cudaStream_t st) {
    Product q{};
    q.a[0] = {p.x, p.x_pitch, 1};
    q.b[0] = {p.w_gate, p.wg_pitch, 1};
    q.b[1] = {p.w_up, p.wu_pitch, 1};
    q.m = p.m, q.n = p.hidden, q.k = p.cin, q.terms = 1;
    q.out = p.a, q.out1 = p.g, q.out2 = p.u, q.pitch = p.h_pitch;
    q.bias0 = p.b_gate, q.bias1 = p.b_up, q.act = p.act;
    FH_TRY((product<T, GLU>(q, st)));
    Product d{};
    d.a[0] = {p.a, p.h_pitch, 1};
    d.b[0] = {p.w_down, p.wd_pitch, 1};
    d.m = p.m, d.n = p.cout, d.k = p.hidden, d.terms = 1;
    d.out = p.y, d.pitch = p.y_pitch, d.bias0 = p.b_down;
    return product<T, PLAIN>(d, st);
}

template <typename T>
cudaError_t gradient(const FhGatedFfnGradParams& p, cudaStream_t st) {
    T* dg = static_cast<T*>(p.scratch);
    T* du = dg + p.m * p.h_pitch;
    Product q{};
    q.a[0] = {p.dy, p.dy_pitch, 1};
    q.b[0] = {p.w_down, 1, p.wd_pitch};
    q.m = p.m, q.n = p.hidden, q.k = p.cout, q.terms = 1;
    q.out = dg, q.out1 = du, q.pitch = p.h_pitch, q.g = p.g, q.u = p.u, q.act = p.act;
    FH_TRY((product<T, GLU_GRAD>(q, st)));
    if (p.dx) {
        Product d{};
        d.a[0] = {dg, p.h_pitch, 1};
        d.a[1] = {du, p.h_pitch, 1};
        d.b[0] = {p.w_gate, 1, p.wg_pitch};
        d.b[1] = {p.w_up, 1, p.wu_pitch};
        d.m = p.m, d.n = p.cin, d.k = p.hidden, d.terms = 2, d.out = p.dx, d.pitch = p.dx_pitch;
        FH_TRY((product<T, PLAIN>(d, st)));
    }
    auto weight = [&](const void* left, long long lp, int n, const void* right, long long rp, int c, void* out,
                      long long op) {
        if (!out) return cudaSuccess;
        Product w{};
        w.a[0] = {left, 1, lp};
        w.b[0] = {right, 1, rp};
        w.m = n, w.n = c, w.k = p.m, w.terms = 1, w.out = out, w.pitch = op;
        return product<T, PLAIN>(w, st);
    };
    FH_TRY(weight(dg, p.h_pitch, p.hidden, p.x, p.x_pitch, p.cin, p.dw_gate, p.dwg_pitch));
    FH_TRY(weight(du, p.h_pitch, p.hidden, p.x, p.x_pitch, p.cin, p.dw_up, p.dwu_pitch));
    FH_TRY(weight(p.dy, p.dy_pitch, p.cout, p.a, p.h_pitch, p.hidden, p.dw_down, p.dwd_pitch));
    if (p.db_gate) FH_TRY(column_sums<T>(dg, p.h_pitch, p.m, p.hidden, p.db_gate, st));
    if (p.db_up) FH_TRY(column_sums<T>(du, p.h_pitch, p.m, p.hidden, p.db_up, st));
    if (p.db_down) FH_TRY(column_sums<T>(p.dy, p.dy_pitch, p.m, p.cout, p.db_down, st));
    return cudaSuccess;
}

}  // namespace

extern "C" size_t fhk_gated_ffn_scratch_bytes(const FhGatedFfnParams* p) {
    (void)p;
    return 0;
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
    if (!p || p->m <= 0 || p->m > kMaxRows || p->h_pitch <= 0) return 0;
    return (size_t)p->m * p->h_pitch * 4;  // dg and du
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

// no waits in this form
extern "C" long long fhk_gated_ffn_wait_timeouts(int) { return 0; }
