// Gated linear layer: [g | u] = x·wᵀ + b, h = act(g)·u, and its backward.
//
//   backward: dg = dh·u·act'(g), du = dh·act(g)
//             dx = [dg|du]·w, dw = [dg|du]ᵀ·x, db = Σ_rows [dg|du]
// h is rounded once from fp32 pre-activations.  [dg|du] is rounded to bf16 for
// dx (a bf16 output); dw is fp32, so there [dg|du] goes in as two bf16 pieces,
// hi = bf16(v) and lo = bf16(v − hi) (2^-18 of v is lost, where one piece loses 2^-9).
#include "gemm_dma.hpp"

namespace {

using namespace nott::gemm;
using nott::ceil_div;
using nott::launch_status;
using nott::WorkspaceHold;

// e^x, the rounding of x·log2 e taken into the result; x within ±126.
__device__ __forceinline__ float exp_near(float x) {
    constexpr float kLog2e = 1.4426950408889634f;
    const float t = x * kLog2e;
    const float r = fmaf(x, kLog2e, -t);
    const float e = __builtin_amdgcn_exp2f(t);
    return fmaf(e, r * 0.69314718f, e);
}
__device__ __forceinline__ float sigmoid(float x) {
    const float e = exp_near(__builtin_amdgcn_fmed3f(-x, -80.f, 80.f));
    return x != x ? x : __builtin_amdgcn_rcpf(1.f + e);
}

// The activation (a) and its derivative (da).
template <int ACT>
__device__ __forceinline__ void activate(float g, float& a, float& da) {
    if constexpr (ACT == NOTT_ACT_SILU) {
        const float e = sigmoid(g);
        a = g * e;
        da = fmaf(a, 1.f - e, e);
    } else if constexpr (ACT == NOTT_ACT_GELU) {
        const float cdf = 0.5f * erfcf(g * -0.70710678f);
        a = g * cdf;
        da = fmaf(g * 0.39894228f, exp_near(fmaxf(-0.5f * g * g, -120.f)), cdf);
    } else if constexpr (ACT == NOTT_ACT_GELU_TANH) {
        const float e = sigmoid(1.5957691f * fmaf(0.044715f * g, g * g, g));
        a = g * e;
        da = fmaf(a * (1.f - e), 1.5957691f * fmaf(0.134145f * g, g, 1.f), e);
    } else if constexpr (ACT == NOTT_ACT_RELU) {
        a = relu_out(g);
        da = g > 0.f ? 1.f : g != g ? g : 0.f;
    } else {
        a = sigmoid(g);
        da = a * (1.f - a);
    }
}

template <class F>
int with_act(int act, F f) {
    switch (act) {
        case NOTT_ACT_SILU: return f(std::integral_constant<int, NOTT_ACT_SILU>());
        case NOTT_ACT_GELU: return f(std::integral_constant<int, NOTT_ACT_GELU>());
        case NOTT_ACT_GELU_TANH: return f(std::integral_constant<int, NOTT_ACT_GELU_TANH>());
        case NOTT_ACT_RELU: return f(std::integral_constant<int, NOTT_ACT_RELU>());
        default: return f(std::integral_constant<int, NOTT_ACT_SIGMOID>());
    }
}

// h (and gu) from the fp32 products pre [m, 2f] and the bias.
template <typename T, int ACT>
__global__ __launch_bounds__(256) void gated_act_kernel(const float* __restrict__ pre, const float* __restrict__ b,
                                                        int64_t m, int64_t f, T* __restrict__ h, T* __restrict__ gu) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= f) return;
    const float bg = b ? b[c] : 0.f, bu = b ? b[f + c] : 0.f;
    for (int64_t r = blockIdx.y; r < m; r += gridDim.y) {
        const float g = pre[r * 2 * f + c] + bg, u = pre[r * 2 * f + f + c] + bu;
        float a, da;
        activate<ACT>(g, a, da);
        Io<T>::st(h, r * f + c, a * u);
        if (gu) {
            Io<T>::st(gu, r * 2 * f + c, g);
            Io<T>::st(gu, r * 2 * f + f + c, u);
        }
    }
}

// [dg|du] [m, 2f] as T, in bf16 also what its rounding leaves (lo).  A workgroup
// takes 64 columns and every gridDim.y-th group of 4 rows; partial (null: no db)
// [gridDim.y][2f] receives its column sums of the unrounded values.
template <typename T, int ACT>
__global__ __launch_bounds__(256) void gated_dact_kernel(const T* __restrict__ dh, const T* __restrict__ gu, int64_t m,
                                                         int64_t f, T* __restrict__ hi, T* __restrict__ lo,
                                                         float* __restrict__ partial) {
    __shared__ float red[2][4][64];
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + lane;
    float sg = 0.f, su = 0.f;
    if (c < f) {
        for (int64_t r = (int64_t)blockIdx.y * 4 + wid; r < m; r += (int64_t)gridDim.y * 4) {
            const float g = Io<T>::ld(gu, r * 2 * f + c), u = Io<T>::ld(gu, r * 2 * f + f + c);
            const float d = Io<T>::ld(dh, r * f + c);
            float a, da;
            activate<ACT>(g, a, da);
            const float dg = d * u * da, du = d * a;
            sg += dg;
            su += du;
            Io<T>::st(hi, r * 2 * f + c, dg);
            Io<T>::st(hi, r * 2 * f + f + c, du);
            if constexpr (sizeof(T) == 2) {
                if (lo) {
                    lo[r * 2 * f + c] = f32_to_bf16(dg - bf16_to_f32(f32_to_bf16(dg)));
                    lo[r * 2 * f + f + c] = f32_to_bf16(du - bf16_to_f32(f32_to_bf16(du)));
                }
            }
        }
    }
    if (!partial) return;
    red[0][wid][lane] = sg;
    red[1][wid][lane] = su;
    __syncthreads();
    if (wid < 2 && c < f)
        partial[(int64_t)blockIdx.y * 2 * f + wid * f + c] =
            (red[wid][0][lane] + red[wid][1][lane]) + (red[wid][2][lane] + red[wid][3][lane]);
}

// db[c] (+)= Σ_z partial[z][c], in z order.
__global__ __launch_bounds__(256) void gated_db_kernel(const float* __restrict__ partial, int slabs, int64_t n,
                                                       float* __restrict__ db, int accumulate) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= n) return;
    float s = 0.f;
#pragma unroll 8
    for (int z = 0; z < slabs; ++z) s += partial[(int64_t)z * n + c];
    db[c] = accumulate ? db[c] + s : s;
}

// dw[o][i] (+)= v.
struct AccStore {
    float* c;
    int64_t M, N;
    int accumulate;
    __device__ __forceinline__ void store(int64_t m, int64_t n, float v) const {
        if (m >= M || n >= N) return;
        float* p = c + m * N + n;
        *p = accumulate ? *p + v : v;
    }
};

// C = A·B, operands as in gemm_dma.hpp, on whichever engine takes them.
template <typename T, bool AT, bool BT, class EP>
int product(nott_ctx ctx, const T* A, int64_t lda, const T* B, int64_t ldb, const EP& ep, int64_t M, int64_t N,
            int64_t K) {
    if constexpr (sizeof(T) == 2) {
        const int st = dma::run<AT, BT>(ctx, A, lda, B, ldb, ep, M, N, K);
        if (st != NOTT_ERR_UNSUPPORTED) return st;
    }
    auto go = [&](const auto& la, const auto& lb) {
        return small_grid(ctx, M, N) ? run_small<T>(ctx, la, lb, ep, M, N, K) : run<T>(ctx, la, lb, ep, M, N, K);
    };
    auto vec = [](const T* p, int64_t ld) { return ((uintptr_t)p % 16) == 0 && (ld * (int64_t)sizeof(T)) % 16 == 0; };
    if constexpr (AT) return go(ColKLoader<T>{A, lda, M, K}, ColKLoader<T>{B, ldb, N, K});
    else if constexpr (BT) return go(RowKLoader<T>{A, lda, M, K, vec(A, lda)}, ColKLoader<T>{B, ldb, N, K});
    else return go(RowKLoader<T>{A, lda, M, K, vec(A, lda)}, RowKLoader<T>{B, ldb, N, K, vec(B, ldb)});
}

template <typename T>
int fwd(nott_ctx ctx, int64_t m, int64_t d, int64_t f, int act, const T* x, const T* w, const float* b, T* h, T* gu) {
    WorkspaceHold ws(ctx, sizeof(float) * (size_t)(m * 2 * f));
    if (!ws.p) return NOTT_ERR_ALLOC;
    float* pre = reinterpret_cast<float*>(ws.p);
    RowMajorStore<float> ep{pre, 2 * f, m, 2 * f, nullptr};
    const int st = product<T, false, false>(ctx, x, d, w, d, ep, m, 2 * f, d);
    if (st != NOTT_OK) return st;
    return with_act(act, [&](auto a) {
        hipLaunchKernelGGL((gated_act_kernel<T, decltype(a)::value>),
                           dim3((unsigned)ceil_div(f, 256), (unsigned)std::min<int64_t>(m, 65535)), dim3(256), 0,
                           ctx->stream, pre, b, m, f, h, gu);
        return launch_status(ctx, "gated_linear");
    });
}

constexpr int kSlabs = 64;

template <typename T>
int bwd(nott_ctx ctx, int64_t m, int64_t d, int64_t f, int act, const T* dh, const T* x, const T* w, const T* gu, T* dx,
        float* dw, float* db, int accumulate) {
    const size_t body = (sizeof(T) * (size_t)(m * 2 * f) + 255) & ~size_t(255);
    const bool two = sizeof(T) == 2 && dw;
    WorkspaceHold ws(ctx, body * (two ? 2 : 1) + (db ? sizeof(float) * kSlabs * 2 * (size_t)f : 0));
    if (!ws.p) return NOTT_ERR_ALLOC;
    T* hi = reinterpret_cast<T*>(ws.p);
    T* lo = two ? reinterpret_cast<T*>(ws.p + body) : nullptr;
    float* partial = db ? reinterpret_cast<float*>(ws.p + body * (two ? 2 : 1)) : nullptr;
    int st = with_act(act, [&](auto a) {
        hipLaunchKernelGGL((gated_dact_kernel<T, decltype(a)::value>), dim3((unsigned)ceil_div(f, 64), kSlabs), dim3(256),
                           0, ctx->stream, dh, gu, m, f, hi, lo, partial);
        return launch_status(ctx, "gated_linear backward");
    });
    if (st != NOTT_OK) return st;
    if (db) {
        hipLaunchKernelGGL(gated_db_kernel, dim3((unsigned)ceil_div(2 * f, 256)), dim3(256), 0, ctx->stream, partial,
                           kSlabs, 2 * f, db, accumulate);
        st = launch_status(ctx, "gated_linear db");
        if (st != NOTT_OK) return st;
    }
    if (dx) {
        RowMajorStore<T> ep{dx, d, m, d, nullptr};
        st = product<T, false, true>(ctx, hi, 2 * f, w, d, ep, m, d, 2 * f);
        if (st != NOTT_OK) return st;
    }
    if (dw) {
        st = product<T, true, true>(ctx, hi, 2 * f, x, d, AccStore{dw, 2 * f, d, accumulate}, 2 * f, d, m);
        if (st != NOTT_OK) return st;
        if (two) st = product<T, true, true>(ctx, lo, 2 * f, x, d, AccStore{dw, 2 * f, d, 1}, 2 * f, d, m);
    }
    return st;
}

}  // namespace

extern "C" int nott_gated_linear_fwd(nott_ctx ctx, nott_dtype dtype, int64_t m, int64_t d, int64_t f, int act,
                                     const void* x, const void* w, const float* b, void* h, void* gu) {
    NOTT_CHECK_CTX(ctx);
    NOTT_REQUIRE(ctx, nott::valid_dtype(dtype), "nott_gated_linear_fwd: bad dtype");
    NOTT_REQUIRE(ctx, act >= NOTT_ACT_SILU && act <= NOTT_ACT_SIGMOID, "nott_gated_linear_fwd: unknown activation");
    NOTT_REQUIRE(ctx, m >= 0 && d > 0 && f > 0, "nott_gated_linear_fwd: need m >= 0, d > 0, f > 0");
    if (m == 0) return NOTT_OK;
    NOTT_REQUIRE(ctx, x && w && h, "nott_gated_linear_fwd: null buffer");
    nott::DeviceScope scope(ctx->device);
    if (dtype == NOTT_F32)
        return fwd<float>(ctx, m, d, f, act, static_cast<const float*>(x), static_cast<const float*>(w), b,
                          static_cast<float*>(h), static_cast<float*>(gu));
    return fwd<bf16_t>(ctx, m, d, f, act, static_cast<const bf16_t*>(x), static_cast<const bf16_t*>(w), b,
                       static_cast<bf16_t*>(h), static_cast<bf16_t*>(gu));
}

extern "C" int nott_gated_linear_bwd(nott_ctx ctx, nott_dtype dtype, int64_t m, int64_t d, int64_t f, int act,
                                     const void* dh, const void* x, const void* w, const void* gu, void* dx, float* dw,
                                     float* db, int accumulate) {
    NOTT_CHECK_CTX(ctx);
    NOTT_REQUIRE(ctx, nott::valid_dtype(dtype), "nott_gated_linear_bwd: bad dtype");
    NOTT_REQUIRE(ctx, act >= NOTT_ACT_SILU && act <= NOTT_ACT_SIGMOID, "nott_gated_linear_bwd: unknown activation");
    NOTT_REQUIRE(ctx, m >= 0 && d > 0 && f > 0, "nott_gated_linear_bwd: need m >= 0, d > 0, f > 0");
    nott::DeviceScope scope(ctx->device);
    if (m == 0) {
        // Empty batch: dx is empty; the parameter gradients sum over nothing.
        if (!accumulate) {
            if (dw && nott_zero(ctx, (int64_t)sizeof(float) * 2 * f * d, dw) != NOTT_OK) return NOTT_ERR_HIP;
            if (db && nott_zero(ctx, (int64_t)sizeof(float) * 2 * f, db) != NOTT_OK) return NOTT_ERR_HIP;
        }
        return NOTT_OK;
    }
    if (!dx && !dw && !db) return NOTT_OK;
    NOTT_REQUIRE(ctx, dh && gu, "nott_gated_linear_bwd: null buffer");
    NOTT_REQUIRE(ctx, !dx || w, "nott_gated_linear_bwd: dx needs w");
    NOTT_REQUIRE(ctx, !dw || x, "nott_gated_linear_bwd: dw needs x");
    if (dtype == NOTT_F32)
        return bwd<float>(ctx, m, d, f, act, static_cast<const float*>(dh), static_cast<const float*>(x),
                          static_cast<const float*>(w), static_cast<const float*>(gu), static_cast<float*>(dx), dw, db,
                          accumulate);
    return bwd<bf16_t>(ctx, m, d, f, act, static_cast<const bf16_t*>(dh), static_cast<const bf16_t*>(x),
                       static_cast<const bf16_t*>(w), static_cast<const bf16_t*>(gu), static_cast<bf16_t*>(dx), dw, db,
                       accumulate);
}
