// Log probabilities of given tokens, with the entropy of each row and its most
// likely tokens, and their gradient.  Per row of logits, z = scale·logit:
//   m = max z, S = Σ exp(z − m), T = Σ exp(z − m)·(z − m)
//   lse = m + log S, logprob = (z_y − m) − log S, entropy = log S − T/S
//   dlogit_j = scale·(dlp·([j = y] − p_j) − dH·p_j·(log p_j + H)), p = exp(z − lse)
// m, S and T are carried together over one read of the row: with a new maximum m'
// and a = exp(m − m'), S' = a·S and T' = a·(T + S·(m − m')).
#include "common.hpp"

namespace {

using nott::ceil_div;

constexpr int64_t kIgnoreIndex = -100;
constexpr int kMaxTop = 64;
constexpr float kLog2e = 1.4426950408889634f;

// e^x for x <= 0: what the rounding of x·log2 e leaves (2^-19 of the result at
// x = −30) is taken into the result.  Below −200 (masked logits: −inf and the
// type's lowest value) 0; NaN stays.
__device__ __forceinline__ float exp_neg(float x) {
    x = x < -200.f ? -200.f : x;
    const float t = x * kLog2e;
    const float r = fmaf(x, kLog2e, -t);
    const float e = __builtin_amdgcn_exp2f(t);
    return fmaf(e, r * 0.69314718f, e);
}

// Logits of −inf or the type's lowest value mask a token: below this there is
// nothing.  As the maximum's first value it keeps −inf − (−inf) out of everything.
constexpr float kNothing = -1e30f;

// The running statistics of a part of a row.  A NaN stays in s and t.
struct Stats {
    float m, s, t;
    __device__ __forceinline__ void add(float z) {
        if (z > m) {
            const float d = m - z, a = exp_neg(d);
            t = a * fmaf(s, fmaxf(d, -200.f), t);
            s *= a;
            m = z;
        }
        const float d = z - m, e = exp_neg(d);
        s += e;
        t = fmaf(e, fmaxf(d, -200.f), t);
    }
    __device__ __forceinline__ void merge(const Stats& o) {
        const float n = fmaxf(m, o.m);
        const float da = m - n, db = o.m - n;
        const float a = exp_neg(da), b = exp_neg(db);
        t = a * fmaf(s, fmaxf(da, -200.f), t) + b * fmaf(o.s, fmaxf(db, -200.f), o.t);
        s = a * s + b * o.s;
        m = n;
    }
};

// Order of the most likely tokens as one whole number: the value in an order that
// integers keep (−0 as +0, NaN above all), then the lower column.
__device__ __forceinline__ uint64_t top_key(float z, uint32_t col) {
    uint32_t u = __builtin_bit_cast(uint32_t, z + 0.f);
    u = z != z ? 0xffffffffu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
    return ((uint64_t)u << 32) | (uint32_t)~col;
}

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int mask) {
    const uint32_t lo = __shfl_xor((uint32_t)v, mask), hi = __shfl_xor((uint32_t)(v >> 32), mask);
    return ((uint64_t)hi << 32) | lo;
}

__device__ __forceinline__ uint64_t block_max64(uint64_t v, uint64_t* red) {
    for (int s = 32; s; s >>= 1) v = max(v, shfl_xor64(v, s));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t r = red[0];
    for (int i = 1; i < (int)blockDim.x / 64; ++i) r = max(r, red[i]);
    __syncthreads();
    return r;
}

struct FwdOut {
    float* logprob;
    float* entropy;
    float* lse;
    float* top_logprob;
    int64_t* top_index;
    unsigned long long* err;
};

// log p of a logit z (scaled) in a row of statistics st.
__device__ __forceinline__ float log_p(float z, const Stats& st, float logs) {
    return st.s == 0.f || z < kNothing ? -INFINITY : (z - st.m) - logs;
}

// The row's outputs from its statistics.
template <typename T>
__device__ __forceinline__ void write_row(const FwdOut& o, int64_t row, int64_t y, int64_t c, const T* z, float scale,
                                          const Stats& st, float logs) {
    const bool empty = st.s == 0.f;   // every token masked
    float lp = 0.f;
    if (y >= 0 && y < c) lp = log_p(Io<T>::ld(z, y) * scale, st, logs);
    else if (y != kIgnoreIndex) atomicAdd(o.err, 1ull);
    o.logprob[row] = lp;
    if (o.lse) o.lse[row] = empty ? -INFINITY : st.m + logs;
    if (o.entropy) o.entropy[row] = empty ? 0.f : logs - st.t / st.s;
}

// Any row, a workgroup each; the top tokens one after the other, each by a scan
// for the largest key below the last one.
template <typename T>
__global__ __launch_bounds__(256) void logprob_any_kernel(const T* __restrict__ logits,
                                                          const int64_t* __restrict__ labels, int64_t c, float scale,
                                                          int top, FwdOut o) {
    __shared__ Stats part[4];
    __shared__ uint64_t red[4];
    const int64_t row = blockIdx.x;
    const T* z = logits + row * c;
    Stats st{kNothing, 0.f, 0.f};
    for (int64_t j = threadIdx.x; j < c; j += 256) st.add(Io<T>::ld(z, j) * scale);
    for (int s = 32; s; s >>= 1) st.merge(Stats{__shfl_xor(st.m, s), __shfl_xor(st.s, s), __shfl_xor(st.t, s)});
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = st;
    __syncthreads();
    st = part[0];
    for (int i = 1; i < 4; ++i) st.merge(part[i]);
    const float logs = logf(st.s);
    if (threadIdx.x == 0) write_row(o, row, labels[row], c, z, scale, st, logs);
    uint64_t last = ~uint64_t(0);
    for (int i = 0; i < top; ++i) {
        uint64_t best = 0;
        for (int64_t j = threadIdx.x; j < c; j += 256) {
            const uint64_t key = top_key(Io<T>::ld(z, j), (uint32_t)j);
            if (key < last && key > best) best = key;
        }
        last = block_max64(best, red);
        if (threadIdx.x == 0) {
            const int64_t j = (uint32_t)~(uint32_t)last;
            o.top_index[row * top + i] = j;
            o.top_logprob[row * top + i] = log_p(Io<T>::ld(z, j) * scale, st, logs);
        }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void logprob_bwd_any_kernel(const T* logits, const int64_t* __restrict__ labels,
                                                              int64_t c, float scale, const float* __restrict__ lse,
                                                              const float* __restrict__ entropy,
                                                              const float* __restrict__ dlogprob,
                                                              const float* __restrict__ dentropy, T* dlogits) {
    const int64_t row = blockIdx.x;
    const int64_t y = labels[row];
    const bool given = y >= 0 && y < c;
    const float l = lse[row], h = dentropy ? entropy[row] : 0.f;
    const float dl = given ? dlogprob[row] : 0.f, dh = dentropy ? dentropy[row] : 0.f;
    for (int64_t j = threadIdx.x; j < c; j += 256) {
        const float lp = Io<T>::ld(logits, row * c + j) * scale - l;
        const float p = exp_neg(lp);
        float g = -p * fmaf(dh, fmaxf(lp, -200.f) + h, dl);
        if (j == y) g += dl;
        Io<T>::st(dlogits, row * c + j, l == -INFINITY ? 0.f : g * scale);
    }
}

}  // namespace

extern "C" int nott_token_logprob_fwd(nott_ctx ctx, nott_dtype dtype, int64_t n, int64_t c, const void* logits,
                                      const int64_t* labels, double scale, int64_t top, float* logprob, float* entropy,
                                      float* lse, float* top_logprob, int64_t* top_index) {
    NOTT_CHECK_CTX(ctx);
    NOTT_REQUIRE(ctx, nott::valid_dtype(dtype), "nott_token_logprob_fwd: bad dtype");
    NOTT_REQUIRE(ctx, n >= 0 && c > 0 && n < (int64_t(1) << 31) && c < (int64_t(1) << 31),
                 "nott_token_logprob_fwd: need 0 <= n and 0 < c, both below 2^31");
    NOTT_REQUIRE(ctx, scale > 0.0 && scale < 1e30, "nott_token_logprob_fwd: scale must be positive and finite");
    NOTT_REQUIRE(ctx, top >= 0 && top <= kMaxTop && top <= c, "nott_token_logprob_fwd: top must be 0 to min(c, 64)");
    if (n == 0) return NOTT_OK;
    NOTT_REQUIRE(ctx, logits && labels && logprob, "nott_token_logprob_fwd: null buffer");
    NOTT_REQUIRE(ctx, top == 0 || (top_logprob && top_index), "nott_token_logprob_fwd: top needs top_logprob and top_index");
    nott::DeviceScope scope(ctx->device);
    const FwdOut o{logprob, entropy, lse, top_logprob, top_index, ctx->err_word};
    if (dtype == NOTT_F32)
        hipLaunchKernelGGL(logprob_any_kernel<float>, dim3((unsigned)n), dim3(256), 0, ctx->stream,
                           static_cast<const float*>(logits), labels, c, (float)scale, (int)top, o);
    else
        hipLaunchKernelGGL(logprob_any_kernel<bf16_t>, dim3((unsigned)n), dim3(256), 0, ctx->stream,
                           static_cast<const bf16_t*>(logits), labels, c, (float)scale, (int)top, o);
    return nott::launch_status(ctx, "token_logprob");
}

extern "C" int nott_token_logprob_bwd(nott_ctx ctx, nott_dtype dtype, int64_t n, int64_t c, const void* logits,
                                      const int64_t* labels, double scale, const float* lse, const float* entropy,
                                      const float* dlogprob, const float* dentropy, void* dlogits) {
    NOTT_CHECK_CTX(ctx);
    NOTT_REQUIRE(ctx, nott::valid_dtype(dtype), "nott_token_logprob_bwd: bad dtype");
    NOTT_REQUIRE(ctx, n >= 0 && c > 0 && n < (int64_t(1) << 31) && c < (int64_t(1) << 31),
                 "nott_token_logprob_bwd: need 0 <= n and 0 < c, both below 2^31");
    NOTT_REQUIRE(ctx, scale > 0.0 && scale < 1e30, "nott_token_logprob_bwd: scale must be positive and finite");
    if (n == 0) return NOTT_OK;
    NOTT_REQUIRE(ctx, logits && labels && lse && dlogprob && dlogits, "nott_token_logprob_bwd: null buffer");
    NOTT_REQUIRE(ctx, !dentropy || entropy, "nott_token_logprob_bwd: dentropy needs entropy");
    nott::DeviceScope scope(ctx->device);
    if (dtype == NOTT_F32)
        hipLaunchKernelGGL(logprob_bwd_any_kernel<float>, dim3((unsigned)n), dim3(256), 0, ctx->stream,
                           static_cast<const float*>(logits), labels, c, (float)scale, lse, entropy, dlogprob, dentropy,
                           static_cast<float*>(dlogits));
    else
        hipLaunchKernelGGL(logprob_bwd_any_kernel<bf16_t>, dim3((unsigned)n), dim3(256), 0, ctx->stream,
                           static_cast<const bf16_t*>(logits), labels, c, (float)scale, lse, entropy, dlogprob, dentropy,
                           static_cast<bf16_t*>(dlogits));
    return nott::launch_status(ctx, "token_logprob backward");
}
