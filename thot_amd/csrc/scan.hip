// Gated linear recurrence over time, forward and backward, channel by channel:
//
//   h_t = keep_t·h_{t−1} + take_t·x_t
//   a = gate or sigmoid(gate);  take = 1 or 1 − a;  keep = a, or 0 where a sequence begins
// backward, with e_t the gradient of h_t and c_t = keep_t·e_t what it hands to t − 1:
//   e_t = dh_t + c_{t+1},  dx = take·e,  da = e·h_{t−1} (0 where a sequence begins) [− e·x]
//
// Composition: a span of tokens maps the state s before it to A·s + B (A = Π keep), and
// two spans in a row to (A₂·A₁, A₂·B₁ + B₂); c is the same recurrence in reverse with the
// same A.  A workgroup owns 32 or 64 channels and takes 256 tokens at a time: each thread
// the span of a few tokens of its channels in registers, all threads fold the spans' maps
// through LDS (the reverse scan's beside), and the spans are gone through again from the
// states before them.  So x and gate are read once and h is written once; the
// backward reads x, gate and dh, forms the states again in fp32 from the one that the
// forward kept before every 256th token (0.8% of h's bytes in bf16, where reading h costs a sixth
// stream and its rounding), and writes dx and dgate.  States, maps and sums are fp32.
//
// Few channels (b·d of a few thousand) do not fill the chip: then the tokens are split
// into segments, whose maps a kernel before forms (reading x and gate once more), and
// each workgroup folds the maps before its segment, in their order.  No workgroup waits
// for another, and results do not depend on timing.
// A keep of exactly 0 forgets the state whatever it was, an infinity or NaN as well.
//
// Bound by HBM (3 streams forward, 5 backward): 4 x 4096 tokens of 2048 channels in bf16
// take 57 us forward (3.6 TB/s) and 97 backward (3.5 TB/s); a packed batch of 50001 tokens
// of 520 channels in fp32 182 us backward (42 of them for the segments' maps; 4.0 TB/s over
// its 7 streams).  A token's row holds 64 to 256 bytes of a workgroup, so neighbouring
// blocks of channels share pages and lines of memory: they run on one XCD, side by side
// (74 us without that, forward; 118 backward).
#include "common.hpp"

#include <type_traits>

namespace {

using nott::ceil_div;

constexpr int kTile = 256;          // tokens of a tile, and between kept states
constexpr int kThreads = 512;

// VEC neighbouring channels of a token: 16 bytes, or one element where rows are not aligned.
template <typename T, int VEC> struct Row;
template <typename T> struct Row<T, 1> {
    typedef T Raw;
    static __device__ __forceinline__ Raw load(const T* p) { return *p; }
    static __device__ __forceinline__ void floats(Raw u, float (&v)[1]) { v[0] = Io<T>::ld(&u, 0); }
    static __device__ __forceinline__ void store(T* p, const float (&v)[1]) { Io<T>::st(p, 0, v[0]); }
};
template <> struct Row<float, 4> {
    typedef f32x4 Raw;
    static __device__ __forceinline__ Raw load(const float* p) { return Pack16<float>::raw(p); }
    static __device__ __forceinline__ void floats(const Raw& u, float (&v)[4]) { Pack16<float>::unpack(u, v); }
    // (a workgroup's 256 bytes of a token are whole lines: past the caches, which then keep inputs)
    static __device__ __forceinline__ void store(float* p, const float (&v)[4]) { Pack16<float>::st<true>(p, v); }
};
template <> struct Row<bf16_t, 8> {
    typedef u32x4 Raw;
    static __device__ __forceinline__ Raw load(const bf16_t* p) { return Pack16<bf16_t>::raw(p); }
    static __device__ __forceinline__ void floats(const Raw& u, float (&v)[8]) { Pack16<bf16_t>::unpack(u, v); }
    static __device__ __forceinline__ void store(bf16_t* p, const float (&v)[8]) { Pack16<bf16_t>::st(p, v); }
};

struct Params {
    int64_t t, seg;                 // tokens, tokens of a segment
    int32_t d, nblk, nseg, nchunk;  // channels, their blocks, segments, kept states
    int64_t rows;                   // b·d
    int64_t xb, xt, gb, gt, hb, ht, dxb, dxt, dgb, dgt;   // batch and token strides
};

// a and 1 − a.  A sigmoid's both come from e^−|g|, so that neither overflows (infinities
// give exactly 0 and 1) and each keeps its bits where it is small.
template <bool SIG>
__device__ __forceinline__ void gates(float g, float& a, float& rest) {
    if constexpr (SIG) {
        const float t = __builtin_amdgcn_exp2f(__builtin_fabsf(g) * -1.4426950f), big = __builtin_amdgcn_rcpf(1.f + t);
        const float small = t * big;
        a = g < 0.f ? small : big;
        rest = g < 0.f ? big : small;
    } else {
        a = g;
        rest = 1.f - g;
    }
}

// A sigmoid is 0 at −infinity alone: where fp32 does not hold it, it is the least number.
template <bool SIG>
__device__ __forceinline__ float opened(float a, float g) {
    return SIG && a == 0.f && g > -INFINITY ? 0x1p-149f : a;
}

// A·s + B; A = 0 forgets s.
__device__ __forceinline__ float step(float A, float s, float B) { return A == 0.f ? B : fmaf(A, s, B); }
__device__ __forceinline__ float step(double A, float s, float B) { return A == 0.0 ? B : (float)fma(A, (double)s, (double)B); }

// Of two maps in a row: 0 where either forgets, beside an infinity or a NaN as well, and only
// there.  A product that fp32 does not hold is its least number (of the product's sign): it
// takes 2^-149 of a state at most in, and leaves one that is infinite or NaN what it is.
__device__ __forceinline__ float both(float A, float B) {
    const float p = A * B;
    const float least = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, p) | 1u);
    return A == 0.f || B == 0.f ? 0.f : p == 0.f ? least : p;
}
// A product over a segment also overflows fp32 (gates above 1 over a thousand tokens, before
// which a state may be 0).  It is formed in fp64, its exponent brought back into ±400 after
// every four gates (2^±149 at most each): a state times that is 0 or infinite in fp32 all the
// same.  An infinite gate's stays infinite, NaN NaN; of a product of 0 the caller takes care.
__device__ __forceinline__ double within(double A) {
    uint64_t bits = __builtin_bit_cast(uint64_t, A);
    const int e = (int)(bits >> 52) & 0x7ff, to = e == 0x7ff ? e : max(1023 - 400, min(1023 + 400, e));
    bits = (bits & ~(uint64_t(0x7ff) << 52)) | (uint64_t)to << 52;
    return __builtin_bit_cast(double, bits);
}

// Keeps the compiler from holding what it formed from x before (an unpacked copy, a
// product) beside x.
template <typename X>
__device__ __forceinline__ void anew(X& x) { asm volatile("" : "+v"(x)); }

// The place of a thread in its workgroup's tile of 256 tokens of CH channels.
template <int VEC, int CH>
struct Place {
    static constexpr int L = CH / VEC, G = kThreads / L, R = kTile / G;   // lanes of a token, spans, tokens of a span
    static constexpr int E = kThreads / CH;                              // threads that fold a channel's maps
    int lane, span, c, cc;          // channels from c; cc: where loads go instead past the end
    int block, seg;                 // of channels; of time
    int64_t b;
    bool in;
    __device__ __forceinline__ explicit Place(const Params& p) {
        // Workgroups are dealt to the 8 XCDs in turn: each XCD takes neighbouring blocks of
        // channels, so that its L2 meets the two halves of a line, and rows near each other.
        const int n = (int)(gridDim.x * gridDim.y), lin = (int)(blockIdx.y * gridDim.x + blockIdx.x);
        const int x = lin & 7, each = n >> 3, more = n & 7;
        int at = x * each + min(x, more) + (lin >> 3);
        seg = at / (int)gridDim.x;
        at -= seg * (int)gridDim.x;
        lane = threadIdx.x % L;
        span = threadIdx.x / L;
        b = at / p.nblk;
        block = at % p.nblk;
        c = block * CH + lane * VEC;
        in = c < p.d;
        cc = in ? c : 0;
    }
};

// Folds the maps of a tile's spans in their order (REVERSE: from the last), by all
// threads: the q-th of E threads of a channel composes its share of the spans (compose),
// then goes through the shares before its own and through its own spans again, and leaves
// in B the state before each (apply): a chain of 31 or fewer steps.
template <int G, int CH, bool REVERSE>
struct Fold {
    static constexpr int E = kThreads / CH, N = G / E;
    float a[N], b[N];
    int q, ch;
    __device__ __forceinline__ Fold() : q(threadIdx.x / CH), ch(threadIdx.x % CH) {}
    __device__ __forceinline__ int span(int i) const { return REVERSE ? G - 1 - (q * N + i) : q * N + i; }
    __device__ __forceinline__ void compose(const float (&A)[G][CH], const float (&B)[G][CH], float (&M)[2][E][CH]) {
        float ca = 1.f, cb = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            a[i] = A[span(i)][ch];
            b[i] = B[span(i)][ch];
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            cb = step(a[i], cb, b[i]);
            ca = both(ca, a[i]);
        }
        M[0][q][ch] = ca;
        M[1][q][ch] = cb;
    }
    // Returns the state behind the spans (in the last share's threads).
    __device__ __forceinline__ float apply(float (&B)[G][CH], const float (&M)[2][E][CH], float s) const {
        float ma[E - 1], mb[E - 1];
#pragma unroll
        for (int j = 0; j < E - 1; ++j) {
            ma[j] = M[0][j][ch];
            mb[j] = M[1][j][ch];
        }
#pragma unroll
        for (int j = 0; j < E - 1; ++j) s = j < q ? step(ma[j], s, mb[j]) : s;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            B[span(i)][ch] = s;
            s = step(a[i], s, b[i]);
        }
        return s;
    }
};

// Maps of whole segments, for the segments that follow (forward) or precede (reverse):
// A in fp64 [nseg][b·d], then B in fp32 [nseg][b·d].  A span is a run of the segment's
// tokens, gone through in registers.
struct Maps {
    double* a;
    float* b;
    // The state behind segment g.
    __device__ __forceinline__ float after(int64_t g, int64_t rows, int64_t row, float s) const {
        return step(a[g * rows + row], s, b[g * rows + row]);
    }
};
template <typename T, int VEC, int CH, bool SIG, bool MIX, bool REVERSE>
__global__ __launch_bounds__(kThreads) void scan_maps_kernel(const T* __restrict__ x, const T* __restrict__ gate,
                                                             const uint8_t* __restrict__ reset, Maps agg, Params p) {
    typedef Place<VEC, CH> P;
    __shared__ __attribute__((aligned(16))) double sA[P::G][CH], mA[P::E][CH];
    __shared__ __attribute__((aligned(16))) float sB[P::G][CH], mB[P::E][CH];
    const P w(p);
    const int seg = REVERSE ? w.seg + 1 : w.seg;
    const int64_t t0 = seg * p.seg, t1 = min(p.t, t0 + p.seg);
    const int64_t run = (p.seg + P::G - 1) / P::G;
    const int64_t r0 = min(t1, t0 + w.span * run), r1 = min(t1, r0 + run);
    const T* px = x + w.b * (REVERSE ? p.hb : p.xb) + w.cc;      // (reverse: dh in x's place)
    const T* pg = gate + w.b * p.gb + w.cc;
    const int64_t xt = REVERSE ? p.ht : p.xt;
    double A[VEC];
    float B[VEC];
    bool forgot[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        A[v] = 1.0;
        B[v] = 0.f;
        forgot[v] = false;
    }
    constexpr int U = VEC == 1 ? 8 : 4;
    for (int64_t q = r0; q < r1; q += U) {
        typename Row<T, VEC>::Raw rx[U], rg[U];
        uint8_t fresh[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t t = REVERSE ? max(r0, r1 - 1 - (q - r0) - u) : min(r1 - 1, q + u);
            rx[u] = Row<T, VEC>::load(px + t * xt);
            rg[u] = Row<T, VEC>::load(pg + t * p.gt);
            fresh[u] = reset ? reset[w.b * p.t + t] : 0;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (q + u >= r1) break;
            float vx[VEC], vg[VEC];
            Row<T, VEC>::floats(rx[u], vx);
            Row<T, VEC>::floats(rg[u], vg);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                float a, rest;
                gates<SIG>(vg[v], a, rest);
                a = fresh[u] ? 0.f : opened<SIG>(a, vg[v]);
                B[v] = REVERSE ? (a == 0.f ? 0.f : a * (vx[v] + B[v])) : step(a, B[v], MIX ? rest * vx[v] : vx[v]);
                A[v] *= (double)a;
                forgot[v] |= a == 0.f;
                if (u % 4 == 3) A[v] = within(A[v]);
            }
        }
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        sA[w.span][w.lane * VEC + v] = forgot[v] ? 0.0 : within(A[v]);
        sB[w.span][w.lane * VEC + v] = B[v];
    }
    __syncthreads();
    // Folded by all threads, as in Fold below: a thread's share of the spans, then the shares.
    constexpr int E = P::E, N = P::G / E;
    const int q = threadIdx.x / CH, c = threadIdx.x % CH, ch = w.block * CH + c;
    double fa;
    float fb;
    auto fold = [&](const auto& a, const auto& b, int first, auto count) {
        double ka[count];
        float kb[count];
#pragma unroll
        for (int i = 0; i < count; ++i) {
            ka[i] = a[REVERSE ? first - i : first + i][c];
            kb[i] = b[REVERSE ? first - i : first + i][c];
        }
        fa = ka[0];
        fb = kb[0];
#pragma unroll
        for (int i = 1; i < count; ++i) {
            fb = step(ka[i], fb, kb[i]);
            fa = fa == 0.0 || ka[i] == 0.0 ? 0.0 : within(fa * ka[i]);
        }
    };
    fold(sA, sB, REVERSE ? P::G - 1 - q * N : q * N, std::integral_constant<int, N>());
    const int share = REVERSE ? E - 1 - q : q;
    mA[share][c] = fa;
    mB[share][c] = fb;
    __syncthreads();
    if (q || ch >= p.d) return;
    fold(mA, mB, REVERSE ? E - 1 : 0, std::integral_constant<int, E>());
    const int64_t at = (int64_t)seg * p.rows + w.b * p.d + ch;
    agg.a[at] = fa;
    agg.b[at] = fb;
}

// (bf16: 128 registers, so that two workgroups share a CU where there are as many: 16 x 1024
// tokens of 2048 channels 51.6 us for 58.4, 1 x 16384 79 for 87; in fp32 and for unaligned
// rows that spills, 79 for 45 and 148 for 75)
template <typename T, int VEC, int CH, bool SIG, bool MIX>
__global__ __launch_bounds__(kThreads, VEC == 8 ? 4 : 2) void scan_fwd_kernel(const T* __restrict__ x, const T* __restrict__ gate,
                                                            const float* __restrict__ h0,
                                                            const uint8_t* __restrict__ reset,
                                                            Maps agg, T* __restrict__ h,
                                                            float* __restrict__ last, float* __restrict__ states, Params p) {
    typedef Place<VEC, CH> P;
    typedef typename Row<T, VEC>::Raw Raw;
    constexpr int R = P::R;
    // two tiles' maps in turn: a tile's are written while another wave still reads the last one's
    __shared__ __attribute__((aligned(16))) float sA[2][P::G][CH], sB[2][P::G][CH];
    __shared__ float sM[2][P::E][CH], carry[2][CH];     // (carry: the state before the tile, and the next one's)
    const P w(p);
    const int seg = w.seg;
    const int64_t t0 = seg * p.seg, t1 = min(p.t, t0 + p.seg);
    const T* px = x + w.b * p.xb + w.cc;
    const T* pg = gate + w.b * p.gb + w.cc;
    T* ph = h + w.b * p.hb + w.cc;
    Fold<P::G, CH, false> fold;
    const int ch = w.block * CH + fold.ch;
    const bool mine = fold.q == 0 && ch < p.d;
    const int64_t row = w.b * p.d + ch;
    if (mine) {
        float s = h0 ? h0[row] : 0.f;
        for (int g = 0; g < seg; ++g) s = agg.after(g, p.rows, row, s);
        carry[0][fold.ch] = s;
    }
    Raw rx[R], rg[R];
    uint32_t fresh = 0;     // bit r: a sequence begins at token r of the span
    auto load = [&](int64_t tile) {
        fresh = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t t = min(p.t - 1, tile + w.span * R + r);
            rx[r] = Row<T, VEC>::load(px + t * p.xt);
            rg[r] = Row<T, VEC>::load(pg + t * p.gt);
            if (reset && reset[w.b * p.t + t]) fresh |= 1u << r;
        }
    };
    load(t0);
    int buf = 0;
    for (int64_t tile = t0; tile < t1; tile += kTile, buf ^= 1) {
        const int live = (int)max<int64_t>(0, min<int64_t>(R, t1 - tile - w.span * R));   // tokens of the span that are there
        float a[R][VEC], u[R][VEC], A[VEC], B[VEC];
        // Where no sequence begins, no token is missing and no gate is 0 (the map's product
        // shows it), the selects of step() and of the tile's end are left out.
        bool careful = reset || tile + kTile > t1;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            A[v] = 1.f;
            B[v] = 0.f;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float vx[VEC], vg[VEC];
            Row<T, VEC>::floats(rx[r], vx);
            Row<T, VEC>::floats(rg[r], vg);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                float rest;
                gates<SIG>(vg[v], a[r][v], rest);
                u[r][v] = MIX ? rest * vx[v] : vx[v];
            }
        }
        if (careful) {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    u[r][v] = r >= live ? 0.f : u[r][v];
                    a[r][v] = r >= live ? 1.f : (fresh >> r) & 1 ? 0.f : a[r][v];
                }
        }
        bool some = false;      // a product of 0, or what an infinity or a NaN made of one
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                B[v] = fmaf(a[r][v], B[v], u[r][v]);
                A[v] *= a[r][v];
            }
            some |= !(__builtin_fabsf(A[v]) > 0.f);
        }
        careful = __any(some);
        if (careful) {
            if (SIG) {
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    float vg[VEC];
                    Row<T, VEC>::floats(rg[r], vg);
#pragma unroll
                    for (int v = 0; v < VEC; ++v)
                        if (!((fresh >> r) & 1)) a[r][v] = opened<SIG>(a[r][v], vg[v]);
                }
            }
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                A[v] = 1.f;
                B[v] = 0.f;
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    B[v] = step(a[r][v], B[v], u[r][v]);
                    A[v] = both(A[v], a[r][v]);
                }
            }
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            sA[buf][w.span][w.lane * VEC + v] = A[v];
            sB[buf][w.span][w.lane * VEC + v] = B[v];
        }
        if (tile + kTile < t1) load(tile + kTile);
        __syncthreads();
        fold.compose(sA[buf], sB[buf], sM);
        __syncthreads();
        {
            const float s = carry[buf][fold.ch];
            if (states && mine) states[(w.b * p.nchunk + tile / kTile) * p.d + ch] = s;
            const float after = fold.apply(sB[buf], sM, s);
            if (fold.q == P::E - 1) carry[buf ^ 1][fold.ch] = after;
        }
        __syncthreads();
        float c[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) c[v] = sB[buf][w.span][w.lane * VEC + v];
        T* po = ph + (tile + w.span * R) * p.ht;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (careful) {
#pragma unroll
                for (int v = 0; v < VEC; ++v) c[v] = step(a[r][v], c[v], u[r][v]);
            } else {
#pragma unroll
                for (int v = 0; v < VEC; ++v) c[v] = fmaf(a[r][v], c[v], u[r][v]);
            }
            if (w.in && r < live) Row<T, VEC>::store(po + r * p.ht, c);
        }
    }
    if (mine && last && t1 == p.t) last[row] = carry[buf][fold.ch];
}

template <typename T, int VEC, int CH, bool SIG, bool MIX>
__global__ __launch_bounds__(kThreads) void scan_bwd_kernel(const T* __restrict__ dh, const T* __restrict__ x,
                                                            const T* __restrict__ gate, const uint8_t* __restrict__ reset,
                                                            const float* __restrict__ states,
                                                            const float* __restrict__ dlast, Maps agg,
                                                            T* __restrict__ dx, T* __restrict__ dgate,
                                                            float* __restrict__ dh0, Params p) {
    typedef Place<VEC, CH> P;
    typedef typename Row<T, VEC>::Raw Raw;
    constexpr int R = P::R;
    // A serves both folds, which run side by side; B and C become the states before a span
    // and the gradients from behind it
    __shared__ __attribute__((aligned(16))) float sA[P::G][CH], sB[P::G][CH], sC[P::G][CH];
    __shared__ float sM[2][2][P::E][CH], carry[2][CH];      // (carry: the gradient from behind the tile)
    const P w(p);
    const int seg = w.seg;
    const int64_t t0 = seg * p.seg, t1 = min(p.t, t0 + p.seg);
    const T* pe = dh + w.b * p.hb + w.cc;
    const T* px = x + w.b * p.xb + w.cc;
    const T* pg = gate + w.b * p.gb + w.cc;
    Fold<P::G, CH, false> states_fold;
    Fold<P::G, CH, true> grads_fold;
    const int fold_ch = states_fold.ch, q = states_fold.q;
    const int ch = w.block * CH + fold_ch;
    const int64_t row = w.b * p.d + ch;
    const bool mine = q == 0 && ch < p.d;
    if (mine) {
        float s = dlast ? dlast[row] : 0.f;
        for (int g = p.nseg - 1; g > seg; --g) s = agg.after(g, p.rows, row, s);
        carry[0][fold_ch] = s;
    }
    int buf = 0;
    Raw re[R], rx[R], rg[R];
    uint32_t fresh = 0;
    auto load = [&](int64_t tile) {
        fresh = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t t = min(p.t - 1, tile + w.span * R + r);
            re[r] = Row<T, VEC>::load(pe + t * p.ht);
            rx[r] = Row<T, VEC>::load(px + t * p.xt);
            rg[r] = Row<T, VEC>::load(pg + t * p.gt);
            if (reset && tile + w.span * R + r < p.t && reset[w.b * p.t + t]) fresh |= 1u << r;
        }
    };
    // Loads of the next tile are in flight while a tile is computed only where both fit the
    // registers.
    constexpr bool AHEAD = VEC == 8;
    const int64_t first = t0, final = t0 + (t1 - t0 - 1) / kTile * kTile;
    if (AHEAD) load(final);
    for (int64_t tile = final; tile >= first; tile -= kTile) {
        if (!AHEAD) load(tile);
        const int live = (int)min<int64_t>(R, t1 - tile - w.span * R);     // tokens of the span that are there
        uint32_t begins = fresh;
        float a[R][VEC], A[VEC], B[VEC], C[VEC];
        float rest[SIG || MIX ? R : 1][VEC];      // 1 − a
        Raw ex[R], ee[R];       // x and dh as loaded: half the registers in bf16
        const float before = ch < p.d ? states[(w.b * p.nchunk + tile / kTile) * p.d + ch] : 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float vg[VEC];
            ex[r] = rx[r];
            ee[r] = re[r];
            Row<T, VEC>::floats(rg[r], vg);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                float rs;
                gates<SIG>(vg[v], a[r][v], rs);
                if constexpr (SIG || MIX) rest[r][v] = rs;
            }
        }
        // The span's maps; CAREFUL as in the forward.
        auto maps = [&](auto which) {
            constexpr bool CAREFUL = decltype(which)::value;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                A[v] = 1.f;
                B[v] = C[v] = 0.f;
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float vx[VEC];
                Row<T, VEC>::floats(ex[r], vx);
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    if (CAREFUL) a[r][v] = r >= live ? 1.f : a[r][v];
                    const float k = CAREFUL && ((begins >> r) & 1) ? 0.f : a[r][v];
                    const float u = CAREFUL && r >= live ? 0.f : MIX ? rest[r][v] * vx[v] : vx[v];
                    B[v] = CAREFUL ? step(k, B[v], u) : fmaf(k, B[v], u);
                    A[v] = CAREFUL ? both(A[v], k) : A[v] * k;
                }
            }
#pragma unroll
            for (int r = R - 1; r >= 0; --r) {
                float ve[VEC];
                Row<T, VEC>::floats(ee[r], ve);
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    const float k = CAREFUL && ((begins >> r) & 1) ? 0.f : a[r][v];
                    const float e = (CAREFUL && r >= live ? 0.f : ve[v]) + C[v];
                    C[v] = CAREFUL && k == 0.f ? 0.f : k * e;
                }
            }
        };
        bool careful = reset || tile + kTile > t1;
        if (!careful) {
            maps(std::false_type());
            bool some = false;
#pragma unroll
            for (int v = 0; v < VEC; ++v) some |= !(__builtin_fabsf(A[v]) > 0.f);
            careful = __any(some);
        }
        if (careful && SIG) {
            bool shut = false;
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int v = 0; v < VEC; ++v) shut |= a[r][v] == 0.f;
            // (in fp32 the gates are read again for it, since no registers are left to keep them:
            // 4 x 4096 tokens of 2048 channels 200 us, 222 with spills)
            if (__any(shut)) {
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    float vg[VEC];
                    Row<T, VEC>::floats(VEC == 4 ? Row<T, VEC>::load(pg + min(p.t - 1, tile + w.span * R + r) * p.gt) : rg[r], vg);
#pragma unroll
                    for (int v = 0; v < VEC; ++v) a[r][v] = opened<SIG>(a[r][v], vg[v]);
                }
            }
        }
        if (careful) maps(std::true_type());
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            sA[w.span][w.lane * VEC + v] = A[v];
            sB[w.span][w.lane * VEC + v] = B[v];
            sC[w.span][w.lane * VEC + v] = C[v];
        }
        if (AHEAD && tile > first) load(tile - kTile);
        __syncthreads();
        states_fold.compose(sA, sB, sM[0]);
        grads_fold.compose(sA, sC, sM[1]);
        __syncthreads();
        (void)states_fold.apply(sB, sM[0], before);
        {
            const float after = grads_fold.apply(sC, sM[1], carry[buf][fold_ch]);
            if (q == P::E - 1) carry[buf ^ 1][fold_ch] = after;
        }
        buf ^= 1;
        __syncthreads();
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            B[v] = sB[w.span][w.lane * VEC + v];
            C[v] = sC[w.span][w.lane * VEC + v];
        }
        __syncthreads();    // the next tile's maps go where these were
        anew(begins);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            anew(ex[r]);
            anew(ee[r]);
        }
        const int64_t mt = tile + w.span * R;
        auto gradients = [&](auto which) {
            constexpr bool CAREFUL = decltype(which)::value;
            float held[R][VEC];     // what e is multiplied by in dgate: the state before the token [− x] [times σ′]
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float vx[VEC];
                Row<T, VEC>::floats(ex[r], vx);
                const bool b = CAREFUL && ((begins >> r) & 1);
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    const float u = MIX ? rest[r][v] * vx[v] : vx[v];
                    held[r][v] = (b ? 0.f : B[v]) - (MIX ? vx[v] : 0.f);
                    if constexpr (SIG) held[r][v] *= a[r][v] * rest[r][v];
                    B[v] = CAREFUL ? step(b ? 0.f : a[r][v], B[v], u) : fmaf(a[r][v], B[v], u);
                }
            }
#pragma unroll
            for (int r = R - 1; r >= 0; --r) {
                float ox[VEC], og[VEC], ve[VEC];
                Row<T, VEC>::floats(ee[r], ve);
                const bool b = CAREFUL && ((begins >> r) & 1);
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    const float k = b ? 0.f : a[r][v];
                    const float e = (CAREFUL && r >= live ? 0.f : ve[v]) + C[v];
                    C[v] = CAREFUL && k == 0.f ? 0.f : k * e;
                    ox[v] = MIX ? rest[r][v] * e : e;
                    og[v] = held[r][v] * e;
                }
                if (w.in && (!CAREFUL || r < live)) {
                    Row<T, VEC>::store(dx + w.b * p.dxb + (mt + r) * p.dxt + w.c, ox);
                    Row<T, VEC>::store(dgate + w.b * p.dgb + (mt + r) * p.dgt + w.c, og);
                }
            }
        };
        if (careful) gradients(std::true_type());
        else gradients(std::false_type());
    }
    if (mine && dh0 && seg == 0) dh0[row] = carry[buf][fold_ch];
}

// Few tokens: a thread goes through them with VEC channels, no tiles (a decoding step of
// 64 x 2048 channels is one read of each input in flight).
template <typename T, int VEC, bool SIG, bool MIX>
__global__ __launch_bounds__(64) void scan_steps_kernel(const T* __restrict__ x, const T* __restrict__ gate,
                                                        const float* __restrict__ h0, const uint8_t* __restrict__ reset,
                                                        T* __restrict__ h, float* __restrict__ last,
                                                        float* __restrict__ states, Params p) {
    const int per = (p.d + VEC - 1) / VEC;
    const int64_t i = (int64_t)blockIdx.x * 64 + threadIdx.x;
    const int64_t b = i / per;
    const int c = (int)(i - b * per) * VEC;
    if (b * p.d >= p.rows) return;
    const int64_t row = b * p.d + c;
    float s[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) s[v] = h0 ? h0[row + v] : 0.f;
    if (states) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) states[row + v] = s[v];
    }
    for (int64_t t = 0; t < p.t; ++t) {
        float vx[VEC], vg[VEC];
        Row<T, VEC>::floats(Row<T, VEC>::load(x + b * p.xb + t * p.xt + c), vx);
        Row<T, VEC>::floats(Row<T, VEC>::load(gate + b * p.gb + t * p.gt + c), vg);
        const bool begins = reset && reset[b * p.t + t];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            float a, rest;
            gates<SIG>(vg[v], a, rest);
            s[v] = step(begins ? 0.f : opened<SIG>(a, vg[v]), s[v], MIX ? rest * vx[v] : vx[v]);
        }
        Row<T, VEC>::store(h + b * p.hb + t * p.ht + c, s);
    }
    if (last) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) last[row + v] = s[v];
    }
}

constexpr int64_t kSteps = 16;      // up to so many tokens the tiles would be nearly empty

// Empty sequences: the state goes through.
__global__ __launch_bounds__(256) void scan_pass_kernel(const float* __restrict__ from, float* __restrict__ to, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n) to[i] = from ? from[i] : 0.f;
}

bool whole(const void* p, int64_t sb, int64_t st, int elem) {
    return (uintptr_t)p % 16 == 0 && sb * elem % 16 == 0 && st * elem % 16 == 0;
}

int check(nott_ctx ctx, const nott_scan_desc* d, nott_dtype dtype, Params* p) {
    NOTT_REQUIRE(ctx, nott::valid_dtype(dtype), "linear scan: bad dtype");
    NOTT_REQUIRE(ctx, d != nullptr, "linear scan: null descriptor");
    NOTT_REQUIRE(ctx, d->b >= 0 && d->t >= 0 && d->d > 0 && d->d < (int64_t(1) << 30) && d->t < (int64_t(1) << 40) &&
                          d->b < (int64_t(1) << 31), "linear scan: bad shape");
    NOTT_REQUIRE(ctx, (d->sigmoid | d->mix) >> 1 == 0, "linear scan: sigmoid and mix are 0 or 1");
    p->t = d->t;
    p->d = (int32_t)d->d;
    p->rows = d->b * d->d;
    p->nchunk = 0;
    NOTT_REQUIRE(ctx, ceil_div(d->t, kTile) < (int64_t(1) << 31) && d->b * ceil_div(d->d, 32) <= 0x7fffffff / 512 &&
                          p->rows < (int64_t(1) << 36), "linear scan: too many channels or tokens");
    p->nchunk = (int32_t)ceil_div(d->t, kTile);
    auto strides = [&](const int64_t (&s)[2], int64_t& sb, int64_t& st) {
        const bool dense = s[0] == 0 && s[1] == 0;
        sb = dense ? d->t * d->d : s[0];
        st = dense ? d->d : s[1];
    };
    strides(d->x_stride, p->xb, p->xt);
    strides(d->gate_stride, p->gb, p->gt);
    strides(d->h_stride, p->hb, p->ht);
    strides(d->dx_stride, p->dxb, p->dxt);
    strides(d->dgate_stride, p->dgb, p->dgt);
    return NOTT_OK;
}

// Segments: one where the channels alone give half of the CUs a workgroup, else as many as
// bring two for each, of about 4 tiles (n tiles make at most n/4 segments, rounded up).
Maps segments(nott_ctx ctx, Params* p, int64_t blocks) {
    const int64_t tiles = p->nchunk;
    int64_t n = blocks >= ctx->num_cu / 2 ? 1 : std::min<int64_t>(ceil_div(2 * ctx->num_cu, blocks), ceil_div(tiles, 4));
    const int64_t len = ceil_div(tiles, n);
    p->seg = len * kTile;
    p->nseg = (int32_t)ceil_div(tiles, len);
    if (p->nseg == 1) return {};
    const int64_t maps = p->nseg * p->rows;
    if (auto* a = static_cast<double*>(nott::optional_workspace(ctx, (size_t)maps * (sizeof(double) + sizeof(float)))))
        return {a, reinterpret_cast<float*>(a + maps)};
    p->nseg = 1;
    p->seg = tiles * kTile;
    return {};
}

// Channels of a workgroup: 64 in fp32 rows of 16-byte groups, else 32, whose half as
// many values a thread leave room for the next tile's loads (4 x 4096 tokens of 2048 channels in
// bf16, forward 66 us with 64 channels and 56 with 32, backward 190 and 98; 50001 tokens of
// 520 channels in fp32, backward 177 and 190).
template <int VEC> constexpr int kChannels = VEC == 4 ? 64 : 32;

template <typename T, int VEC, bool SIG, bool MIX>
int fwd(nott_ctx ctx, Params& p, const void* x, const void* gate, const float* h0, const uint8_t* reset, void* h,
        float* last, float* states) {
    const T* tx = static_cast<const T*>(x);
    const T* tg = static_cast<const T*>(gate);
    const int64_t batches = p.rows / p.d;
    if (p.t <= kSteps) {
        const int64_t n = batches * ceil_div(p.d, VEC);
        hipLaunchKernelGGL((scan_steps_kernel<T, VEC, SIG, MIX>), dim3((unsigned)ceil_div(n, 64)), dim3(64), 0, ctx->stream, tx,
                           tg, h0, reset, static_cast<T*>(h), last, states, p);
        return nott::launch_status(ctx, "scan_steps_kernel");
    }
    constexpr int CH = kChannels<VEC>;
    p.nblk = (int32_t)ceil_div(p.d, CH);
    const Maps agg = segments(ctx, &p, batches * p.nblk);
    const dim3 grid((unsigned)(batches * p.nblk));
    if (p.nseg > 1)
        hipLaunchKernelGGL((scan_maps_kernel<T, VEC, CH, SIG, MIX, false>), dim3(grid.x, (unsigned)(p.nseg - 1)), dim3(kThreads),
                           0, ctx->stream, tx, tg, reset, agg, p);
    hipLaunchKernelGGL((scan_fwd_kernel<T, VEC, CH, SIG, MIX>), dim3(grid.x, (unsigned)p.nseg), dim3(kThreads), 0, ctx->stream,
                       tx, tg, h0, reset, agg, static_cast<T*>(h), last, states, p);
    return nott::launch_status(ctx, "scan_fwd_kernel");
}

template <typename T, int VEC, bool SIG, bool MIX>
int bwd(nott_ctx ctx, Params& p, const void* dh, const void* x, const void* gate, const uint8_t* reset, const float* states,
        const float* dlast, void* dx, void* dgate, float* dh0) {
    const T* te = static_cast<const T*>(dh);
    const T* tg = static_cast<const T*>(gate);
    constexpr int CH = kChannels<VEC>;
    p.nblk = (int32_t)ceil_div(p.d, CH);
    const Maps agg = segments(ctx, &p, p.rows / p.d * p.nblk);
    const dim3 grid((unsigned)(p.rows / p.d * p.nblk));
    if (p.nseg > 1)
        hipLaunchKernelGGL((scan_maps_kernel<T, VEC, CH, SIG, false, true>), dim3(grid.x, (unsigned)(p.nseg - 1)),
                           dim3(kThreads), 0, ctx->stream, te, tg, reset, agg, p);
    hipLaunchKernelGGL((scan_bwd_kernel<T, VEC, CH, SIG, MIX>), dim3(grid.x, (unsigned)p.nseg), dim3(kThreads), 0, ctx->stream,
                       te, static_cast<const T*>(x), tg, reset, states, dlast, agg, static_cast<T*>(dx),
                       static_cast<T*>(dgate), dh0, p);
    return nott::launch_status(ctx, "scan_bwd_kernel");
}

// Calls f with the type, width and gate form as template arguments.
template <typename F>
int dispatch(nott_dtype dtype, bool wide, const nott_scan_desc* d, F&& f) {
    auto gate = [&](auto t, auto vec) {
        using std::bool_constant;
        if (d->sigmoid) return d->mix ? f(t, vec, bool_constant<true>(), bool_constant<true>())
                                      : f(t, vec, bool_constant<true>(), bool_constant<false>());
        return d->mix ? f(t, vec, bool_constant<false>(), bool_constant<true>())
                      : f(t, vec, bool_constant<false>(), bool_constant<false>());
    };
    if (dtype == NOTT_BF16)
        return wide ? gate(bf16_t(), std::integral_constant<int, 8>()) : gate(bf16_t(), std::integral_constant<int, 1>());
    return wide ? gate(float(), std::integral_constant<int, 4>()) : gate(float(), std::integral_constant<int, 1>());
}

}  // namespace

extern "C" int nott_linear_scan_fwd(nott_ctx ctx, const nott_scan_desc* d, nott_dtype dtype, const void* x, const void* gate,
                                    const float* h0, const uint8_t* reset, void* h, float* last, float* states) {
    NOTT_CHECK_CTX(ctx);
    Params p{};
    if (const int st = check(ctx, d, dtype, &p); st != NOTT_OK) return st;
    if (p.rows == 0) return NOTT_OK;
    nott::DeviceScope scope(ctx->device);
    if (p.t == 0) {
        if (last)
            hipLaunchKernelGGL(scan_pass_kernel, dim3((unsigned)ceil_div(p.rows, 256)), dim3(256), 0, ctx->stream, h0, last, p.rows);
        return nott::launch_status(ctx, "scan_pass_kernel");
    }
    NOTT_REQUIRE(ctx, x && gate && h, "nott_linear_scan_fwd: null buffer");
    const int elem = (int)nott::dtype_size(dtype);
    const bool wide = whole(x, p.xb, p.xt, elem) && whole(gate, p.gb, p.gt, elem) && whole(h, p.hb, p.ht, elem) &&
                      p.d * elem % 16 == 0;
    return dispatch(dtype, wide, d, [&](auto t, auto vec, auto sig, auto mix) {
        return fwd<decltype(t), decltype(vec)::value, decltype(sig)::value, decltype(mix)::value>(ctx, p, x, gate, h0, reset, h,
                                                                                                  last, states);
    });
}

extern "C" int nott_linear_scan_bwd(nott_ctx ctx, const nott_scan_desc* d, nott_dtype dtype, const void* dh, const void* x,
                                    const void* gate, const uint8_t* reset, const float* states, const float* dlast, void* dx,
                                    void* dgate, float* dh0) {
    NOTT_CHECK_CTX(ctx);
    Params p{};
    if (const int st = check(ctx, d, dtype, &p); st != NOTT_OK) return st;
    if (p.rows == 0) return NOTT_OK;
    nott::DeviceScope scope(ctx->device);
    if (p.t == 0) {
        if (dh0)
            hipLaunchKernelGGL(scan_pass_kernel, dim3((unsigned)ceil_div(p.rows, 256)), dim3(256), 0, ctx->stream, dlast, dh0, p.rows);
        return nott::launch_status(ctx, "scan_pass_kernel");
    }
    NOTT_REQUIRE(ctx, dh && x && gate && states && dx && dgate, "nott_linear_scan_bwd: null buffer");
    const int elem = (int)nott::dtype_size(dtype);
    const bool wide = whole(x, p.xb, p.xt, elem) && whole(gate, p.gb, p.gt, elem) && whole(dh, p.hb, p.ht, elem) &&
                      whole(dx, p.dxb, p.dxt, elem) && whole(dgate, p.dgb, p.dgt, elem) && p.d * elem % 16 == 0;
    return dispatch(dtype, wide, d, [&](auto t, auto vec, auto sig, auto mix) {
        return bwd<decltype(t), decltype(vec)::value, decltype(sig)::value, decltype(mix)::value>(
            ctx, p, dh, x, gate, reset, states, dlast, dx, dgate, dh0);
    });
}
