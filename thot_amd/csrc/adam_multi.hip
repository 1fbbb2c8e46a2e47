// Adam / AdamW over many tensors where they lie, moments in 32 or in 8 bits.
//
// The update is adam.hip's, element by element:
//   m = β1·m + (1−β1)·g,  v = β2·v + (1−β2)·g²,  p −= lr/bc1 · m / (sqrt(v)/sqrt(bc2) + eps)
// with weight decay as there.  With 32-bit moments the results are the bits of
// nott_adam_step.
//
// 8-bit moments.  Blocks of 256 elements hold m and r = sqrt(v) as e4m3 codes (OCP: 4
// exponent and 3 mantissa bits, largest value 448) times an fp32 scale each,
// scale = max |·| / 448.  The root is what the update divides by, so its rounding (2^-4
// at most) is the update's, and its range of 2.3e5 within a block is 5e10 of v.  The
// scale is not rounded to a power of two: a block whose gradients fade decays by β
// through its scale, while codes alone would stay where they are (β2's step of 0.1% is far
// below half a code).  A root above zero never gets the code of zero, which would
// divide m by eps alone; it takes the least code.  The update itself uses m and r in fp32,
// before they are rounded, and the hardware's reciprocal (1 ulp).
//
// Moments of either width are whole blocks of 256; what lies behind a tensor's end is
// updated as elements without a gradient.
// One launch takes up to kTensors tensors of one pair of types: their descriptors are
// kernel arguments (no table in memory to keep or to upload, and a captured graph holds
// them), a workgroup finds its tensor by bisection.  A half-wave owns a block of 256
// (8 elements a lane), so the maxima are five exchanges in registers.
// Bound by HBM: 18 B a parameter with fp32 p, g, a bf16 copy and 8-bit moments, 10 B with
// bf16 p and g, 28 B with fp32 and 32-bit moments.
#include "adam.hpp"

namespace {

using namespace nott::adam;

constexpr int kBlock = 256;                 // elements that share a scale
constexpr int kThreads = 256;               // 8 blocks at a time
constexpr int kUnroll = 2;
constexpr int kChunk = kThreads * 8 * kUnroll;   // elements a workgroup takes
constexpr int kTensors = 56;                // 3.7 KB of kernel arguments

struct Entry {
    void* p;
    void* g;
    void* m;
    void* v;
    float* scale;       // {m's, r's} of each block (8-bit moments)
    bf16_t* copy;       // nullable
    int64_t n;
    int32_t first;      // its first workgroup
    int32_t vec;        // p, g and copy take vector accesses
};
struct Args {
    Entry e[kTensors];
    AdamScalars s;
    const AdamScalars* sdev;
    const float* gscale;
    int32_t count, mode, zero, reserved;
};
static_assert(sizeof(Args) <= 4096, "kernel arguments");

// Lane l of a half-wave (0..31) holds elements 4l..4l+3 and 128 + 4l.. of its block, so
// that each 16-byte access of fp32 lies next to its neighbour's.
__device__ __forceinline__ int place(int l, int half) { return 128 * half + 4 * l; }

// Four elements: as loaded, and as floats.  WHOLE: the workgroup's elements are all
// there and aligned; else element by element.
template <typename T> struct Four;
template <> struct Four<float> {
    typedef f32x4 Raw;
    static __device__ __forceinline__ f32x4 floats(Raw u) { return u; }
    static __device__ __forceinline__ Raw raw(f32x4 v) { return v; }
};
template <> struct Four<bf16_t> {
    typedef u32x2 Raw;
    static __device__ __forceinline__ f32x4 floats(Raw u) {
        return f32x4{__builtin_bit_cast(float, u.x << 16), __builtin_bit_cast(float, u.x & 0xffff0000u),
                     __builtin_bit_cast(float, u.y << 16), __builtin_bit_cast(float, u.y & 0xffff0000u)};
    }
    static __device__ __forceinline__ Raw raw(f32x4 v) { return u32x2{pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w)}; }
};
template <typename T, bool WHOLE>
__device__ __forceinline__ typename Four<T>::Raw load4(const T* p, int64_t i, int64_t n) {
    typedef typename Four<T>::Raw Raw;
    if constexpr (WHOLE) return __builtin_nontemporal_load(reinterpret_cast<const Raw*>(p + i));
    f32x4 r = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (i + e < n) r[e] = Io<T>::ld(p, i + e);
    return Four<T>::raw(r);
}
template <typename T, bool WHOLE>
__device__ __forceinline__ void store4(T* p, int64_t i, int64_t n, f32x4 v) {
    typedef typename Four<T>::Raw Raw;
    if constexpr (WHOLE) {
        __builtin_nontemporal_store(Four<T>::raw(v), reinterpret_cast<Raw*>(p + i));
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (i + e < n) Io<T>::st(p, i + e, v[e]);
}

// Four e4m3 codes of a word as floats, and back (round to nearest even; |v| ≤ 448).
__device__ __forceinline__ f32x4 from_e4m3(uint32_t w) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return f32x4{a.x, a.y, b.x, b.y};
}
__device__ __forceinline__ uint32_t to_e4m3(f32x4 v) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(v.x, v.y, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(v.z, v.w, w, true);
    return (uint32_t)w;
}

// Maximum over a half-wave, in every lane of it.
__device__ __forceinline__ float half_wave_max(float v) {
    v = fmaxf(v, dpp_f32<0xB1>(v));
    v = fmaxf(v, dpp_f32<0x4E>(v));
    v = fmaxf(v, dpp_f32<0x141>(v));
    v = fmaxf(v, dpp_f32<0x140>(v));
    return fmaxf(v, __shfl_xor(v, 16, 64));
}

// 1/scale of a block whose largest magnitude is `top`; a block below 2^-112 counts as zero
// (its inverse would leave fp32's range).
__device__ __forceinline__ float inverse_scale(float top, float& scale) {
    scale = top * (1.f / 448.f);
    const bool some = top >= 0x1p-112f;     // (false for NaN, which fmaxf drops)
    scale = some ? scale : 0.f;
    return some ? 1.f / scale : 0.f;
}

// a·x + b·y with each product rounded: a moment's bits, and so its code, do not depend on
// which of the products a compiler fuses.
__device__ __forceinline__ float mix(float x, float a, float y, float b) {
#pragma clang fp contract(off)
    return x * a + y * b;
}

template <typename TP, typename TG, int BITS, bool WHOLE>
__device__ __forceinline__ void update(const Args& a, const Entry& e, const AdamScalars& s, float gs, int64_t base) {
    TP* p = static_cast<TP*>(e.p);
    TG* g = static_cast<TG*>(e.g);
    uint8_t* m8 = static_cast<uint8_t*>(e.m);
    uint8_t* r8 = static_cast<uint8_t*>(e.v);
    float* m32 = static_cast<float*>(e.m);
    float* v32 = static_cast<float*>(e.v);
    const int l = threadIdx.x & 31;
    typename Four<TP>::Raw pr[kUnroll][2];
    typename Four<TG>::Raw gr[kUnroll][2];
    f32x4 mf[kUnroll][2], vf[kUnroll][2];
    uint32_t mc[kUnroll][2], vc[kUnroll][2];
    f32x2 sc[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int64_t b0 = base + (int64_t)u * (kThreads * 8);
        if (!WHOLE && b0 >= e.n) break;
        // (the moments are whole blocks)
        if constexpr (BITS == 8) sc[u] = *reinterpret_cast<const f32x2*>(e.scale + 2 * (b0 / kBlock));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t i = b0 + place(l, h);
            pr[u][h] = load4<TP, WHOLE>(p, i, e.n);
            gr[u][h] = load4<TG, WHOLE>(g, i, e.n);
            if constexpr (BITS == 8) {
                mc[u][h] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(m8 + i));
                vc[u][h] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(r8 + i));
            } else {
                mf[u][h] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(m32 + i));
                vf[u][h] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(v32 + i));
            }
        }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int64_t b0 = base + (int64_t)u * (kThreads * 8);
        if (!WHOLE && b0 >= e.n) break;
        f32x4 pv[2];
        if constexpr (BITS == 8) {
            const float rbc2 = 1.f / s.bc2_sqrt;
            float mtop = 0.f, rtop = 0.f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const f32x4 mq = from_e4m3(mc[u][h]), rq = from_e4m3(vc[u][h]), gv = Four<TG>::floats(gr[u][h]);
                pv[h] = Four<TP>::floats(pr[u][h]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float pe = pv[h][j], ge = gv[j] * gs;
                    if (a.mode == 2) pe *= s.decay;
                    if (a.mode == 1) ge = fmaf(pe, s.wd, ge);
                    const float m = mf[u][h][j] = mix(mq[j] * sc[u].x, s.beta1, ge, s.one_m_b1);
                    const float r0 = rq[j] * sc[u].y;
                    const float r = vf[u][h][j] = __builtin_sqrtf(mix(r0 * r0, s.beta2, ge * ge, s.one_m_b2));
                    pv[h][j] = fmaf(s.neg_step * m, __builtin_amdgcn_rcpf(fmaf(r, rbc2, s.eps)), pe);
                    mtop = fmaxf(mtop, __builtin_fabsf(m));
                    rtop = fmaxf(rtop, r);
                }
            }
            float ms, rs;
            const float mi = inverse_scale(half_wave_max(mtop), ms), ri = inverse_scale(half_wave_max(rtop), rs);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int64_t i = b0 + place(l, h);
                f32x4 mq, rq;       // at most 448 + an ulp, which rounds to 448; NaN keeps a code of its own
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float r = vf[u][h][j], q = r * ri;
                    mq[j] = mf[u][h][j] * mi;
                    rq[j] = r > 0.f && q < 0x1p-9f ? 0x1p-9f : q;
                }
                __builtin_nontemporal_store(to_e4m3(mq), reinterpret_cast<uint32_t*>(m8 + i));
                __builtin_nontemporal_store(to_e4m3(rq), reinterpret_cast<uint32_t*>(r8 + i));
            }
            if (l == 0) *reinterpret_cast<f32x2*>(e.scale + 2 * (b0 / kBlock)) = f32x2{ms, rs};
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int64_t i = b0 + place(l, h);
                const f32x4 gv = Four<TG>::floats(gr[u][h]);
                pv[h] = Four<TP>::floats(pr[u][h]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float pe = pv[h][j], me = mf[u][h][j], ve = vf[u][h][j];
                    const float ge = gv[j] * gs;
                    if (a.mode == 2) adam_elem<2>(pe, ge, me, ve, s);
                    else if (a.mode == 1) adam_elem<1>(pe, ge, me, ve, s);
                    else adam_elem<0>(pe, ge, me, ve, s);
                    pv[h][j] = pe;
                    mf[u][h][j] = me;
                    vf[u][h][j] = ve;
                }
                __builtin_nontemporal_store(mf[u][h], reinterpret_cast<f32x4*>(m32 + i));
                __builtin_nontemporal_store(vf[u][h], reinterpret_cast<f32x4*>(v32 + i));
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t i = b0 + place(l, h);
            store4<TP, WHOLE>(p, i, e.n, pv[h]);
            if (e.copy) store4<bf16_t, WHOLE>(e.copy, i, e.n, pv[h]);
            if (a.zero) store4<TG, WHOLE>(g, i, e.n, f32x4{0.f, 0.f, 0.f, 0.f});
        }
    }
}

template <typename TP, typename TG, int BITS>
__global__ __launch_bounds__(kThreads) void adam_multi_kernel(Args a) {
    // the tensor whose workgroups include this one
    int lo = 0, hi = a.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.e[mid].first <= (int)blockIdx.x) lo = mid;
        else hi = mid - 1;
    }
    const Entry e = a.e[lo];
    const AdamScalars s = a.sdev ? *a.sdev : a.s;
    const float gs = a.gscale ? *a.gscale : 1.f;
    const int64_t chunk = (int64_t)((int)blockIdx.x - e.first) * kChunk;
    const int64_t base = chunk + (threadIdx.x >> 5) * kBlock;
    if (e.vec && chunk + kChunk <= e.n) update<TP, TG, BITS, true>(a, e, s, gs, base);
    else update<TP, TG, BITS, false>(a, e, s, gs, base);
}

bool aligned(const void* p, size_t to) { return (uintptr_t)p % to == 0; }

int check(nott_ctx ctx, const nott_adam_tensor* t, int64_t count) {
    NOTT_REQUIRE(ctx, count >= 0 && (count == 0 || t), "adam over tensors: bad list");
    for (int64_t i = 0; i < count; ++i) {
        const nott_adam_tensor& x = t[i];
        // (its workgroups' threads fit a launch)
        NOTT_REQUIRE(ctx, x.n >= 0 && x.n <= (int64_t)(0x7fffffff / kThreads) * kChunk, "adam over tensors: bad size");
        NOTT_REQUIRE(ctx, nott::valid_dtype(x.p_dtype) && nott::valid_dtype(x.g_dtype) && (x.bits == 8 || x.bits == 32),
                     "adam over tensors: bad dtype or moments that are not 8 or 32 bits");
        if (x.n == 0) continue;
        NOTT_REQUIRE(ctx, x.p && x.g && x.m && x.v && (x.bits == 32 || x.scale), "adam over tensors: null buffer");
        NOTT_REQUIRE(ctx, aligned(x.p, nott::dtype_size((nott_dtype)x.p_dtype)) &&
                              aligned(x.g, nott::dtype_size((nott_dtype)x.g_dtype)) && aligned(x.copy, 2),
                     "adam over tensors: a misaligned buffer");
        NOTT_REQUIRE(ctx, aligned(x.m, 16) && aligned(x.v, 16) && (x.bits == 32 || aligned(x.scale, 8)),
                     "adam over tensors: moments must be 16-byte aligned, scales 8-byte");
    }
    return NOTT_OK;
}

// Launches for the tensors of one pair of types, kTensors at a time.
template <typename TP, typename TG, int BITS>
int launch(nott_ctx ctx, const nott_adam_tensor* t, int64_t count, Args& a) {
    constexpr int tp = sizeof(TP) == 2 ? NOTT_BF16 : NOTT_F32, tg = sizeof(TG) == 2 ? NOTT_BF16 : NOTT_F32;
    int64_t chunks = 0;
    a.count = 0;
    auto flush = [&]() {
        if (a.count) {
            hipLaunchKernelGGL((adam_multi_kernel<TP, TG, BITS>), dim3((unsigned)chunks), dim3(kThreads), 0, ctx->stream, a);
            a.count = 0;
            chunks = 0;
            return nott::launch_status(ctx, "adam_multi_kernel");
        }
        return (int)NOTT_OK;
    };
    for (int64_t i = 0; i < count; ++i) {
        const nott_adam_tensor& x = t[i];
        if (x.n == 0 || x.p_dtype != tp || x.g_dtype != tg || x.bits != BITS) continue;
        const int64_t mine = nott::ceil_div(x.n, kChunk);
        if (a.count == kTensors || chunks + mine > 0x7fffffff / kThreads)   // the launch's threads fit 31 bits
            if (const int st = flush(); st != NOTT_OK) return st;
        a.e[a.count++] = {x.p, x.g, x.m, x.v, x.scale, static_cast<bf16_t*>(x.copy), x.n, (int32_t)chunks,
                          aligned(x.p, 4 * sizeof(TP)) && aligned(x.g, 4 * sizeof(TG)) && aligned(x.copy, 8)};
        chunks += mine;
    }
    return flush();
}

int run(nott_ctx ctx, const nott_adam_tensor* t, int64_t count, Args& a) {
    auto types = [&](auto bits) {
        constexpr int B = decltype(bits)::value;
        int st = launch<float, float, B>(ctx, t, count, a);
        if (st == NOTT_OK) st = launch<bf16_t, bf16_t, B>(ctx, t, count, a);
        if (st == NOTT_OK) st = launch<float, bf16_t, B>(ctx, t, count, a);
        return st == NOTT_OK ? launch<bf16_t, float, B>(ctx, t, count, a) : st;
    };
    const int st = types(std::integral_constant<int, 8>());
    return st == NOTT_OK ? types(std::integral_constant<int, 32>()) : st;
}

}  // namespace

extern "C" int nott_adam_multi_step(nott_ctx ctx, int decoupled, const nott_adam_tensor* tensors, int64_t count, double lr,
                                    double beta1, double beta2, double eps, double weight_decay, int64_t step,
                                    const float* grad_scale, int zero_grad_after) {
    NOTT_CHECK_CTX(ctx);
    if (const int st = check(ctx, tensors, count); st != NOTT_OK) return st;
    NOTT_REQUIRE(ctx, step >= 1, "nott_adam_multi_step: step must be >= 1 (post-increment count)");
    NOTT_REQUIRE(ctx, lr >= 0.0 && eps >= 0.0 && weight_decay >= 0.0, "nott_adam_multi_step: negative lr/eps/weight_decay");
    NOTT_REQUIRE(ctx, beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0,
                 "nott_adam_multi_step: betas must be in [0, 1)");
    nott::DeviceScope scope(ctx->device);
    Args a{};
    a.s = make_scalars(lr, beta1, beta2, eps, weight_decay, step);
    a.mode = weight_decay == 0.0 ? 0 : (decoupled ? 2 : 1);
    a.gscale = grad_scale;
    a.zero = zero_grad_after != 0;
    return run(ctx, tensors, count, a);
}

extern "C" int nott_adam_multi_step_graph(nott_ctx ctx, int decoupled, const nott_adam_tensor* tensors, int64_t count,
                                          const double* hparams, nott_adam_device_state* state, int weight_decay_nonzero,
                                          const float* grad_scale, int zero_grad_after) {
    NOTT_CHECK_CTX(ctx);
    if (const int st = check(ctx, tensors, count); st != NOTT_OK) return st;
    NOTT_REQUIRE(ctx, hparams && state, "nott_adam_multi_step_graph: null hyper-parameters or state");
    nott::DeviceScope scope(ctx->device);
    hipLaunchKernelGGL(adam_prep_kernel, dim3(1), dim3(1), 0, ctx->stream, hparams, state);
    Args a{};
    a.sdev = reinterpret_cast<const AdamScalars*>(state->reserved);
    a.mode = !weight_decay_nonzero ? 0 : (decoupled ? 2 : 1);
    a.gscale = grad_scale;
    a.zero = zero_grad_after != 0;
    return run(ctx, tensors, count, a);
}
