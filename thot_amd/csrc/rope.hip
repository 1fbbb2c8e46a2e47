// Queries and keys between the packed projection and attention: root-mean-square
// norm of every head, its weight, and the rotation by position, one pass.
//
//   forward : z = x·r·γ, r = 1/sqrt(mean x² + eps);  y = R(θ)·z
//   backward: dz = R(θ)ᵀ·dy;  x̂ = x·r
//             dx = r·(γ·dz − x̂·mean(γ·dz·x̂)),  dγ = Σ_{tokens, heads} dz·x̂
// R turns the pairs (a, b) of the first `rot` elements by θ = position·inv_freq.
// All arithmetic is fp32 on values rounded once, at the store; the angle is
// taken in 64 bits as a fraction of a turn and reduced to [-1/2, 1/2] before it
// is rounded, so that far positions (θ of 1e5 and more) keep their last bits.
#include "common.hpp"

namespace {

using nott::ceil_div;

constexpr int kMaxHead = 512;
constexpr int kMaxAxes = 4;

// Positions and frequencies; pair i belongs to the axis whose `first` is the last <= i.
struct Turns {
    const int64_t* positions;
    const double* inv_freq;
    int64_t tokens;
    int32_t first[kMaxAxes];   // past the axes: rot/2
    int32_t half;              // rot/2
    int32_t interleaved;
    __device__ __forceinline__ int64_t position(int64_t token, int pair) const {
        int axis = 0;
#pragma unroll
        for (int a = 1; a < kMaxAxes; ++a) axis += pair >= first[a] ? 1 : 0;
        return positions[axis * tokens + token];
    }
    __device__ __forceinline__ void turn(int64_t token, int pair, float& c, float& s) const {
        // 1/(2π) in two parts: the second keeps what is left of a turn right past
        // angles of 2^29, where the first's rounding reaches fp32
        constexpr double kTurn = 0x1.45f306dc9c883p-3, kTurnLow = -0x1.6b01ec5417056p-57;
        const double angle = (double)position(token, pair) * inv_freq[pair];
        const double r = fma(angle, kTurn, -rint(angle * kTurn)) + angle * kTurnLow;
        sincospif(2.f * (float)r, &s, &c);
    }
};

// One of the two tensors: its heads, input x, output gradient dy (backward),
// output, and their strides {batch, token, head}.
template <typename T>
struct Heads {
    const T* x;
    const T* dy;
    T* out;
    const T* gamma;
    int64_t xs[3], ys[3], os[3];
    int32_t n;
};

template <typename T>
struct RopeArgs {
    Heads<T> q, k;
    Turns turns;
    int32_t t, dh, norm;
    float eps;
    FastDiv by_heads, by_t, by_width;   // by_width: pairs of a token's table
    float* partial;     // backward: [grid][2·dh] sums of dz·x̂, q then k; null: not asked for
};

__device__ __forceinline__ int64_t at(const int64_t (&s)[3], uint32_t b, uint32_t t, uint32_t h) {
    return b * s[0] + t * s[1] + h * s[2];
}

// Any head size, alignment and number of rotated elements: a wave per head, element
// e = 64·v + lane, the other element of its pair by a second load (from the caches).
// As in rope_vec_kernel a workgroup takes `tpb` tokens and forms their cosines and
// sines once, in LDS; a wave has U heads in flight.  Every load of a head comes
// before its stores (the stores wait for the loaded values), so an output may be
// its input.  Bound by instructions (one element a lane): 2x4096 tokens, 16+16 heads
// of 64, rot 36, bf16 58 us forward, 118 backward; the kernel below takes 15.6 and 31
// with rot 64.
template <typename T, int V, bool BWD>
__global__ __launch_bounds__(256) void rope_any_kernel(RopeArgs<T> a, int tpb) {
    constexpr int U = V <= 2 ? 4 : V == 4 ? 2 : 1;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    f32x2* table = reinterpret_cast<f32x2*>(lds);   // [tpb][rot/2] {cos, sin}
    const int tid = (int)threadIdx.x, lane = tid & 63, wid = tid >> 6;
    const int half = a.turns.half, heads = a.q.n + a.k.n;
    const bool inter = a.turns.interleaved;
    // of each element: its pair's other one (itself past the rotated ones), which of
    // the two it is, its pair, and both weights
    int other[V], pair[V];
    bool second[V];
    float g[2][V], go[2][V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int e = min(64 * v + lane, a.dh - 1);
        const bool rotated = e < 2 * half;
        second[v] = rotated && (inter ? (e & 1) != 0 : e >= half);
        other[v] = !rotated ? e : inter ? e ^ 1 : second[v] ? e - half : e + half;
        pair[v] = !rotated ? -1 : inter ? e >> 1 : second[v] ? e - half : e;
        g[0][v] = a.q.gamma ? Io<T>::ld(a.q.gamma, e) : 1.f;
        g[1][v] = a.k.gamma ? Io<T>::ld(a.k.gamma, e) : 1.f;
        go[0][v] = a.q.gamma ? Io<T>::ld(a.q.gamma, other[v]) : 1.f;
        go[1][v] = a.k.gamma ? Io<T>::ld(a.k.gamma, other[v]) : 1.f;
    }
    float dg[2][V];
#pragma unroll
    for (int v = 0; v < V; ++v) dg[0][v] = dg[1][v] = 0.f;
    const bool has_x = !BWD || a.norm;
    for (int64_t t0 = (int64_t)blockIdx.x * tpb; t0 < a.turns.tokens; t0 += (int64_t)gridDim.x * tpb) {
        const int nt = (int)min((int64_t)tpb, a.turns.tokens - t0), items = nt * heads;
        if (half > 0) {
            __syncthreads();   // the last tokens' readers are done
            for (int i = tid; i < nt * half; i += 256) {
                const int t = i / half;
                float c, s;
                a.turns.turn(t0 + t, i - t * half, c, s);
                table[i] = f32x2{c, s};
            }
            __syncthreads();
        }
        for (int base = wid * U; base < items; base += 4 * U) {
            float xv[U][V], xo[U][V], dv[U][V], dn[U][V];
            T* out[U];
            int tok[U], side[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                uint32_t t, head, bi, ti;
                a.by_heads.divmod((uint32_t)min(base + u, items - 1), t, head);
                a.by_t.divmod((uint32_t)t0 + t, bi, ti);
                tok[u] = (int)t;
                side[u] = head < (uint32_t)a.q.n ? 0 : 1;
                const Heads<T>& h = side[u] ? a.k : a.q;
                if (side[u]) head -= a.q.n;
                const T* x = h.x + (has_x ? at(h.xs, bi, ti, head) : 0);
                const T* dy = BWD ? h.dy + at(h.ys, bi, ti, head) : nullptr;
                out[u] = h.out + (BWD ? at(h.os, bi, ti, head) : at(h.ys, bi, ti, head));
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const int e = min(64 * v + lane, a.dh - 1);
                    xv[u][v] = has_x ? Io<T>::ld(x, e) : 0.f;
                    if constexpr (!BWD) {
                        xo[u][v] = Io<T>::ld(x, other[v]);
                    } else {
                        dv[u][v] = Io<T>::ld(dy, e);
                        dn[u][v] = Io<T>::ld(dy, other[v]);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float ss = 0.f, r = 1.f, dot = 0.f, ov[V];
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (64 * v + lane < a.dh) ss = fmaf(xv[u][v], xv[u][v], ss);
                if (a.norm) r = rsqrtf(wave_sum(ss) / (float)a.dh + a.eps);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    float c = 1.f, s = 0.f;
                    if (pair[v] >= 0) {
                        const f32x2 cs = table[tok[u] * half + pair[v]];
                        c = cs.x;
                        s = second[v] != BWD ? cs.y : -cs.y;
                    }
                    const float gm = side[u] ? g[1][v] : g[0][v];
                    if constexpr (!BWD) {
                        const float w = side[u] ? go[1][v] : go[0][v];
                        const float z = a.norm ? xv[u][v] * r * gm : xv[u][v];
                        const float zo = a.norm ? xo[u][v] * r * w : xo[u][v];
                        ov[v] = pair[v] < 0 ? z : fmaf(zo, s, z * c);   // unrotated: as it is, infinities too
                    } else {
                        const float dz = pair[v] < 0 ? dv[u][v] : fmaf(dn[u][v], s, dv[u][v] * c), xh = xv[u][v] * r;
                        if (base + u < items) {
                            if (side[u]) dg[1][v] = fmaf(dz, xh, dg[1][v]);
                            else dg[0][v] = fmaf(dz, xh, dg[0][v]);
                        }
                        ov[v] = a.norm ? dz * gm : dz;
                        if (64 * v + lane < a.dh) dot = fmaf(ov[v], xh, dot);
                    }
                }
                if constexpr (BWD) {
                    if (a.norm) {
                        dot = wave_sum(dot) / (float)a.dh;
#pragma unroll
                        for (int v = 0; v < V; ++v) ov[v] = r * (ov[v] - xv[u][v] * r * dot);
                    }
                }
                if (base + u < items) {
#pragma unroll
                    for (int v = 0; v < V; ++v)
                        if (64 * v + lane < a.dh) Io<T>::st(out[u], 64 * v + lane, ov[v]);
                }
            }
        }
    }
    if constexpr (BWD) {
        if (!a.partial) return;
        __syncthreads();
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (64 * v + lane < a.dh) {
                lds[wid * 2 * a.dh + 64 * v + lane] = dg[0][v];
                lds[(wid * 2 + 1) * a.dh + 64 * v + lane] = dg[1][v];
            }
        __syncthreads();
        float* p = a.partial + (int64_t)blockIdx.x * 2 * a.dh;
        for (int j = tid; j < 2 * a.dh; j += 256)
            p[j] = (lds[j] + lds[2 * a.dh + j]) + (lds[4 * a.dh + j] + lds[6 * a.dh + j]);
    }
}

// Σ over the LPH lanes (a power of two) that share a head; all of them get it.
template <int LPH>
__device__ __forceinline__ float head_sum(float v) {
    if constexpr (LPH >= 2) v += dpp_f32<0xB1>(v);    // quad_perm [1,0,3,2]
    if constexpr (LPH >= 4) v += dpp_f32<0x4E>(v);    // quad_perm [2,3,0,1]
    if constexpr (LPH >= 8) v += dpp_f32<0x141>(v);   // row_half_mirror
    if constexpr (LPH >= 16) v += dpp_f32<0x140>(v);  // row_mirror
    if constexpr (LPH >= 32) v += __shfl_xor(v, 16);
    if constexpr (LPH >= 64) v += __shfl_xor(v, 32);
    return v;
}

template <typename T>
__device__ __forceinline__ typename Pack16<T>::Raw ones() {
    if constexpr (sizeof(T) == 2) return u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
    else return f32x4{1.f, 1.f, 1.f, 1.f};
}

// Heads of whole aligned 16-byte chunks: LPH lanes a head, each with two chunks
// that hold both elements of its pairs (chunks c and c + rot/2, or neighbours), so
// a head's norm, weight and rotation need no exchange but the sum.  A workgroup
// takes `tpb` tokens at a time: it issues the loads of its first heads, forms the
// tokens' cosines and sines in LDS while they are on their way (once for all
// heads), then runs over the heads, U in flight a lane.
// Memory bound: one read and one write of q and k (and one more read backward).
// 8x1024 tokens, 16+16 heads of 64, bf16: 15.6 us forward (4.3 TB/s), 2x4096 tokens,
// 24+4 heads of 128 25.8 (4.6), fp32 42.7 (5.5); backward of 4x4096 tokens, 32+8
// heads of 128, bf16 118 us (4.3 TB/s).  Three backward workgroups a CU (a register
// limit of 168) against two: video in fp32 41 -> 31 us.
template <typename T, int LPH, bool BWD>
__global__ __launch_bounds__(256, BWD ? 3 : 1) void rope_vec_kernel(RopeArgs<T> a, int tpb) {
    constexpr int E = Pack16<T>::N, GPB = 256 / LPH, U = BWD ? 2 : 4;
    typedef typename Pack16<T>::Raw Raw;
    // {cos, sin} of each token's pairs, two pairs (16 bytes) of every chunk side by
    // side: [tpb][pairs of a chunk / 2][chunks], so that the lanes of a head read a
    // run.  Half-split: a chunk of E pairs for each rotated lane; neighbours: a
    // chunk's E/2 pairs, those past the rotated ones with the angle 0.
    extern __shared__ __attribute__((aligned(16))) float lds[];
    f32x4* table = reinterpret_cast<f32x4*>(lds);
    const int tid = (int)threadIdx.x, slot = tid % LPH, group = tid / LPH;
    const int half = a.turns.half, nc = a.dh / E, heads = a.q.n + a.k.n;
    const bool inter = a.turns.interleaved;
    // this lane's chunks; rotated: they are the two halves of pairs
    const int hc = inter ? 0 : half / E;
    const bool rotated = slot < hc;
    const int c0 = rotated ? slot : 2 * hc + 2 * (slot - hc), c1 = rotated ? slot + hc : c0 + 1;
    const bool has0 = c0 < nc, has1 = c1 < nc;
    const int n0 = half - c0 * (E / 2), n1 = half - c1 * (E / 2);   // neighbours: rotated pairs from each chunk's start on
    const int e0 = has0 ? c0 * E : 0, e1 = has1 ? c1 * E : 0;
    const int ppc = inter ? E / 2 : E, chunks = inter ? nc : hc, width = ppc * chunks;   // of a token's table
    const float inv_dh = 1.f / (float)a.dh;
    const Raw one = ones<T>();
    const Raw gq0 = a.q.gamma ? Pack16<T>::raw(a.q.gamma + e0) : one, gq1 = a.q.gamma ? Pack16<T>::raw(a.q.gamma + e1) : one;
    const Raw gk0 = a.k.gamma ? Pack16<T>::raw(a.k.gamma + e0) : one, gk1 = a.k.gamma ? Pack16<T>::raw(a.k.gamma + e1) : one;
    float dg[BWD ? 4 : 1][E];   // dγ of this lane's chunks: q, q, k, k
#pragma unroll
    for (auto& d : dg)
#pragma unroll
        for (int e = 0; e < E; ++e) d[e] = 0.f;
    for (int64_t t0 = (int64_t)blockIdx.x * tpb; t0 < a.turns.tokens; t0 += (int64_t)gridDim.x * tpb) {
        const int nt = (int)min((int64_t)tpb, a.turns.tokens - t0);
        const int items = nt * heads;
        for (int base = 0; base < items; base += GPB * U) {
            Raw rx[U][2], rd[BWD ? U : 1][2];
            int64_t to[U];
            uint32_t tok[U];
            bool of_q[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                uint32_t head, bi, ti;
                a.by_heads.divmod((uint32_t)min(base + u * GPB + group, items - 1), tok[u], head);
                a.by_t.divmod((uint32_t)t0 + tok[u], bi, ti);
                of_q[u] = head < (uint32_t)a.q.n;
                if (!of_q[u]) head -= a.q.n;
                const Heads<T>& h = of_q[u] ? a.q : a.k;
                if (!BWD || a.norm) {
                    const T* x = h.x + at(h.xs, bi, ti, head);
                    rx[u][0] = Pack16<T>::raw(x + e0);
                    rx[u][1] = Pack16<T>::raw(x + e1);
                }
                if constexpr (BWD) {
                    const T* dy = h.dy + at(h.ys, bi, ti, head);
                    rd[u][0] = Pack16<T>::raw(dy + e0);
                    rd[u][1] = Pack16<T>::raw(dy + e1);
                }
                to[u] = BWD ? at(h.os, bi, ti, head) : at(h.ys, bi, ti, head);
            }
            if (base == 0 && half > 0) {
                __syncthreads();   // the last tokens' readers are done
                for (int i = tid; i < nt * width; i += 256) {
                    uint32_t t, pair;
                    a.by_width.divmod((uint32_t)i, t, pair);
                    float c = 1.f, s = 0.f;
                    if ((int)pair < half) a.turns.turn(t0 + t, (int)pair, c, s);
                    const int chunk = (int)pair / ppc, in = (int)pair % ppc;
                    reinterpret_cast<f32x2*>(lds)[t * width + ((in >> 1) * chunks + chunk) * 2 + (in & 1)] = f32x2{c, s};
                }
                __syncthreads();
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float v0[E], v1[E];
                const f32x4* tab = table + (int)tok[u] * (width / 2);
                // turns the pair (a, b) by {cos, sin}, BWD: back
                auto turn2 = [](float& a, float& b, float c, float s, bool on = true) {
                    if (BWD) s = -s;
                    const float y = fmaf(-b, s, a * c);
                    b = on ? fmaf(a, s, b * c) : b;
                    a = on ? y : a;
                };
                auto turn = [&](float (&p)[E], float (&q)[E]) {
                    if (half == 0) return;
                    if (!inter) {
                        if (!rotated) return;
#pragma unroll
                        for (int e = 0; e < E; e += 2) {
                            const f32x4 cs = tab[e / 2 * chunks + c0];
                            turn2(p[e], q[e], cs.x, cs.y);
                            turn2(p[e + 1], q[e + 1], cs.z, cs.w);
                        }
                        return;
                    }
#pragma unroll
                    for (int e = 0; e < E; e += 4) {
                        const f32x4 cs = tab[e / 4 * chunks + (has0 ? c0 : 0)], ct = tab[e / 4 * chunks + (has1 ? c1 : 0)];
                        // past the rotated pairs as they are (an infinity times a sine of 0 is NaN)
                        turn2(p[e], p[e + 1], cs.x, cs.y, e / 2 < n0);
                        turn2(p[e + 2], p[e + 3], cs.z, cs.w, e / 2 + 1 < n0);
                        turn2(q[e], q[e + 1], ct.x, ct.y, e / 2 < n1);
                        turn2(q[e + 2], q[e + 3], ct.z, ct.w, e / 2 + 1 < n1);
                    }
                };
                float x0[E], x1[E], r = 1.f;
                if (!BWD || a.norm) {
                    // absent chunks are zero
                    Pack16<T>::unpack(has0 ? rx[u][0] : Raw{}, x0);
                    Pack16<T>::unpack(has1 ? rx[u][1] : Raw{}, x1);
                    float ss = 0.f;
#pragma unroll
                    for (int e = 0; e < E; ++e) ss = fmaf(x0[e], x0[e], fmaf(x1[e], x1[e], ss));
                    if (a.norm) r = rsqrtf(fmaf(head_sum<LPH>(ss), inv_dh, a.eps));
                }
                float g0[E], g1[E];
                Pack16<T>::unpack(of_q[u] ? gq0 : gk0, g0);
                Pack16<T>::unpack(of_q[u] ? gq1 : gk1, g1);
                if constexpr (!BWD) {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        v0[e] = a.norm ? x0[e] * r * g0[e] : x0[e];
                        v1[e] = a.norm ? x1[e] * r * g1[e] : x1[e];
                    }
                    turn(v0, v1);
                } else {
                    Pack16<T>::unpack(rd[u][0], v0);
                    Pack16<T>::unpack(rd[u][1], v1);
                    turn(v0, v1);
                    if (a.norm) {
                        // an item past the last adds nothing to dγ
                        const bool counts = base + u * GPB + group < items;
                        float dot = 0.f;
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            x0[e] *= r;
                            x1[e] *= r;
                        }
                        if (counts && of_q[u]) {
#pragma unroll
                            for (int e = 0; e < E; ++e) {
                                dg[0][e] = fmaf(v0[e], x0[e], dg[0][e]);
                                dg[1][e] = fmaf(v1[e], x1[e], dg[1][e]);
                            }
                        } else if (counts) {
#pragma unroll
                            for (int e = 0; e < E; ++e) {
                                dg[2][e] = fmaf(v0[e], x0[e], dg[2][e]);
                                dg[3][e] = fmaf(v1[e], x1[e], dg[3][e]);
                            }
                        }
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            v0[e] *= g0[e];
                            v1[e] *= g1[e];
                            dot = fmaf(v0[e], x0[e], fmaf(v1[e], x1[e], dot));
                        }
                        dot = head_sum<LPH>(dot) * inv_dh;
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            v0[e] = r * fmaf(-x0[e], dot, v0[e]);
                            v1[e] = r * fmaf(-x1[e], dot, v1[e]);
                        }
                    }
                }
                if (base + u * GPB + group < items) {
                    T* out = (of_q[u] ? a.q.out : a.k.out) + to[u];
                    if (has0) Pack16<T>::st(out + e0, v0);
                    if (has1) Pack16<T>::st(out + e1, v1);
                }
            }
        }
    }
    if constexpr (BWD) {
        if (!a.partial) return;
        // over the wave's heads, then the four waves in order
        __syncthreads();
        const int lane = tid & 63, wid = tid >> 6;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e) {
#pragma unroll
                for (int s = LPH; s < 64; s <<= 1) dg[i][e] += __shfl_xor(dg[i][e], s);
                if (lane < LPH && ((i & 1) ? has1 : has0))
                    lds[(wid * 2 + (i >> 1)) * a.dh + ((i & 1) ? e1 : e0) + e] = dg[i][e];
            }
        __syncthreads();
        float* p = a.partial + (int64_t)blockIdx.x * 2 * a.dh;
        for (int j = tid; j < 2 * a.dh; j += 256)
            p[j] = (lds[j] + lds[2 * a.dh + j]) + (lds[4 * a.dh + j] + lds[6 * a.dh + j]);
    }
}

// dγ (+)= Σ_blocks partial[block], in an order that the grid alone fixes: a
// workgroup has 16 columns, 64 threads of each taking every 64th block.
__global__ __launch_bounds__(1024) void rope_dgamma_kernel(const float* __restrict__ partial, int blocks, int dh,
                                                           float* __restrict__ dgq, float* __restrict__ dgk,
                                                           int accumulate) {
    __shared__ float red[64][17];
    const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
    const int col = blockIdx.x * 16 + c, at = col < 2 * dh ? col : 0;
    red[r][c] = r < blocks ? ordered_sum1(partial + (int64_t)r * 2 * dh + at, (int64_t)64 * 2 * dh, (blocks - r + 63) / 64) : 0.f;
    __syncthreads();
    if (r != 0 || col >= 2 * dh) return;
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 64; ++i) t += red[i][c];
    float* out = col < dh ? dgq : dgk;
    if (!out) return;
    const int e = col < dh ? col : col - dh;
    out[e] = accumulate ? out[e] + t : t;
}

// `given`, or the strides of a contiguous [b, t, h, dh] where they are all 0.
void strides(const int64_t (&given)[3], int64_t t, int64_t h, int64_t dh, int64_t (&s)[3]) {
    const bool dense = given[0] == 0 && given[1] == 0 && given[2] == 0;
    s[0] = dense ? t * h * dh : given[0];
    s[1] = dense ? h * dh : given[1];
    s[2] = dense ? dh : given[2];
}

int check(nott_ctx ctx, const nott_qk_rope_desc* d, nott_dtype dtype, const char* who) {
    auto bad = [&](const char* what) { return nott::fail(ctx, NOTT_ERR_INVALID_ARG, std::string(who) + ": " + what); };
    if (!d) return bad("null descriptor");
    if (!nott::valid_dtype(dtype)) return bad("bad dtype");
    if (d->b < 0 || d->t < 0 || d->hq < 0 || d->hk < 0) return bad("negative size");
    if (d->dh < 1 || d->dh > kMaxHead) return bad("head size must be 1 to 512");
    if (d->rot < 0 || d->rot > d->dh || d->rot % 2) return bad("rot must be even, 0 to the head size");
    if (d->axes < 1 || d->axes > kMaxAxes) return bad("axes must be 1 to 4");
    int64_t pairs = 0;
    for (int i = 0; i < kMaxAxes; ++i) {
        if (d->section[i] < 0 || d->section[i] > d->rot || (i >= d->axes && d->section[i] != 0)) return bad("bad section");
        pairs += d->section[i];
    }
    if (pairs != d->rot / 2) return bad("sections must add up to rot/2");
    if (d->norm != 0 && d->norm != 1) return bad("norm must be 0 or 1");
    if (!(d->eps >= 0.0)) return bad("eps must not be negative");
    if (d->hq > 65535 || d->hk > 65535) return bad("too many heads");
    const int64_t most = (int64_t(1) << 31) - 1;
    if (d->b > most || d->t > most || (d->t && d->b > most / d->t) ||
        (d->hq + d->hk && d->b * d->t > most / (d->hq + d->hk)))
        return bad("too many tokens times heads");
    return NOTT_OK;
}

// Pairs of a token's cosine and sine table: the head's where pairs are neighbours.
template <typename T>
int table_pairs(const RopeArgs<T>& a) {
    return a.turns.half == 0 ? 0 : a.turns.interleaved ? a.dh / 2 : a.turns.half;
}

template <typename T>
RopeArgs<T> make_args(const nott_qk_rope_desc& d, const void* q, const void* k, const void* dyq, const void* dyk,
                      const void* gq, const void* gk, const int64_t* positions, const double* inv_freq, void* oq,
                      void* ok) {
    RopeArgs<T> a{};
    auto side = [&](Heads<T>& h, const void* x, const void* dy, void* out, const void* g, int64_t n,
                    const int64_t (&xs)[3], const int64_t (&ys)[3], const int64_t (&os)[3]) {
        h.x = static_cast<const T*>(x);
        h.dy = static_cast<const T*>(dy);
        h.out = static_cast<T*>(out);
        h.gamma = static_cast<const T*>(g);
        h.n = (int32_t)n;
        strides(xs, d.t, n, d.dh, h.xs);
        strides(ys, d.t, n, d.dh, h.ys);
        strides(os, d.t, n, d.dh, h.os);
    };
    side(a.q, q, dyq, oq, gq, d.hq, d.q_stride, d.yq_stride, d.dq_stride);
    side(a.k, k, dyk, ok, gk, d.hk, d.k_stride, d.yk_stride, d.dk_stride);
    a.turns.positions = positions;
    a.turns.inv_freq = inv_freq;
    a.turns.tokens = d.b * d.t;
    a.turns.half = (int32_t)(d.rot / 2);
    a.turns.interleaved = d.interleaved != 0;
    int64_t first = 0;
    for (int i = 0; i < kMaxAxes; ++i) {
        a.turns.first[i] = i < d.axes ? (int32_t)first : a.turns.half;
        first += d.section[i];
    }
    a.t = (int32_t)d.t;
    a.dh = (int32_t)d.dh;
    a.norm = d.norm;
    a.eps = (float)d.eps;
    a.by_heads = FastDiv((uint32_t)(d.hq + d.hk));
    a.by_t = FastDiv((uint32_t)d.t);
    a.by_width = FastDiv((uint32_t)std::max<int64_t>(1, table_pairs(a)));
    return a;
}

// Whether the heads are whole 16-byte chunks wherever they lie, and no chunk holds
// both rotated halves.
template <typename T>
bool in_chunks(const RopeArgs<T>& a, bool bwd) {
    constexpr int E = Pack16<T>::N;
    if (a.dh % E || (!a.turns.interleaved && a.turns.half % E)) return false;
    for (const Heads<T>* h : {&a.q, &a.k}) {
        if (h->n == 0) continue;
        const bool x = !bwd || a.norm;
        for (const void* p : {(const void*)(x ? h->x : nullptr), (const void*)h->dy, (const void*)h->out, (const void*)h->gamma})
            if ((uintptr_t)p % 16) return false;
        for (int i = 0; i < 3; ++i)
            if ((x && h->xs[i] % E) || h->ys[i] % E || (bwd && h->os[i] % E)) return false;
    }
    return true;
}

struct Launch {
    unsigned grid;
    int lph, tpb;
    size_t lds;
};
// Tokens that a workgroup takes at a time: forward as many as fill its lanes' loads
// once; backward, where each workgroup leaves partial sums of dγ, its share of the
// 3 workgroups a CU that its registers allow (fp32 4: 77 against 80 us at 2x4096
// tokens, 24+4 heads of 128; bf16 53 against 47).  Fewer where there are too few for every CU, and with at most
// 16 KiB of cosines and sines.
template <typename T>
Launch plan(nott_ctx ctx, const RopeArgs<T>& a, bool bwd, bool vec) {
    constexpr int E = Pack16<T>::N, kGroups = sizeof(T) == 2 ? 3 : 4;
    Launch l{};
    const int slots = (a.dh / E + 1) / 2, pairs = vec ? table_pairs(a) : a.turns.half;
    if (vec)
        for (l.lph = 2; l.lph < slots;) l.lph *= 2;
    else
        l.lph = 64;
    const int64_t tokens = a.turns.tokens, groups = kGroups * (int64_t)ctx->num_cu;
    int64_t tpb = bwd ? ceil_div(tokens, groups) : (int64_t)(256 / l.lph) * 4 / (a.q.n + a.k.n);
    if (pairs) tpb = std::min<int64_t>(tpb, 2048 / pairs);
    tpb = std::min<int64_t>(tpb, ceil_div(tokens, ctx->num_cu));
    l.tpb = (int)std::max<int64_t>(tpb, 1);
    l.grid = (unsigned)std::min<int64_t>(ceil_div(tokens, l.tpb), bwd ? groups : 1 << 23);   // a launch's threads in 32 bits
    l.lds = std::max(sizeof(f32x2) * (size_t)l.tpb * pairs, bwd ? sizeof(float) * 8 * (size_t)a.dh : 0);
    return l;
}

template <typename T, bool BWD>
void launch_vec(nott_ctx ctx, const Launch& l, const RopeArgs<T>& a) {
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(l.grid), dim3(256), l.lds, ctx->stream, a, l.tpb); };
    switch (l.lph) {
        case 2: return go(rope_vec_kernel<T, 2, BWD>);
        case 4: return go(rope_vec_kernel<T, 4, BWD>);
        case 8: return go(rope_vec_kernel<T, 8, BWD>);
        case 16: return go(rope_vec_kernel<T, 16, BWD>);
        case 32: return go(rope_vec_kernel<T, 32, BWD>);
        default:   // fp32 heads past 256
            if constexpr (sizeof(T) == 4) return go(rope_vec_kernel<T, 64, BWD>);
    }
}

template <typename T, bool BWD>
void launch_any(nott_ctx ctx, const Launch& l, const RopeArgs<T>& a) {
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(l.grid), dim3(256), l.lds, ctx->stream, a, l.tpb); };
    if (a.dh <= 64) go(rope_any_kernel<T, 1, BWD>);
    else if (a.dh <= 128) go(rope_any_kernel<T, 2, BWD>);
    else if (a.dh <= 256) go(rope_any_kernel<T, 4, BWD>);
    else go(rope_any_kernel<T, 8, BWD>);
}

template <typename T>
int forward(nott_ctx ctx, const RopeArgs<T>& a) {
    const bool vec = in_chunks(a, false);
    const Launch l = plan(ctx, a, false, vec);
    if (vec) launch_vec<T, false>(ctx, l, a);
    else launch_any<T, false>(ctx, l, a);
    return nott::launch_status(ctx, "qk_norm_rope");
}

template <typename T>
int backward(nott_ctx ctx, RopeArgs<T> a, float* dgq, float* dgk, int accumulate) {
    const bool vec = in_chunks(a, true);
    const Launch l = plan(ctx, a, true, vec);
    if (a.norm && (dgq || dgk)) {
        a.partial = static_cast<float*>(nott::workspace(ctx, sizeof(float) * 2 * (size_t)a.dh * l.grid));
        if (!a.partial) return NOTT_ERR_ALLOC;
    }
    if (vec) launch_vec<T, true>(ctx, l, a);
    else launch_any<T, true>(ctx, l, a);
    if (a.partial)
        hipLaunchKernelGGL(rope_dgamma_kernel, dim3((unsigned)ceil_div(2 * a.dh, 16)), dim3(1024), 0, ctx->stream,
                           a.partial, (int)l.grid, a.dh, dgq, dgk, accumulate);
    return nott::launch_status(ctx, "qk_norm_rope backward");
}

}  // namespace

extern "C" int nott_qk_norm_rope_fwd(nott_ctx ctx, const nott_qk_rope_desc* d, nott_dtype dtype, const void* q,
                                     const void* k, const void* gamma_q, const void* gamma_k, const int64_t* positions,
                                     const double* inv_freq, void* yq, void* yk) {
    NOTT_CHECK_CTX(ctx);
    const int st = check(ctx, d, dtype, "nott_qk_norm_rope_fwd");
    if (st != NOTT_OK) return st;
    if (d->b * d->t * (d->hq + d->hk) == 0) return NOTT_OK;
    NOTT_REQUIRE(ctx, (d->hq == 0 || (q && yq)) && (d->hk == 0 || (k && yk)), "nott_qk_norm_rope_fwd: null buffer");
    NOTT_REQUIRE(ctx, d->rot == 0 || (positions && inv_freq), "nott_qk_norm_rope_fwd: null positions or inv_freq");
    NOTT_REQUIRE(ctx, d->norm || (!gamma_q && !gamma_k), "nott_qk_norm_rope_fwd: a weight needs the norm");
    nott::DeviceScope scope(ctx->device);
    if (dtype == NOTT_F32)
        return forward(ctx, make_args<float>(*d, q, k, nullptr, nullptr, gamma_q, gamma_k, positions, inv_freq, yq, yk));
    return forward(ctx, make_args<bf16_t>(*d, q, k, nullptr, nullptr, gamma_q, gamma_k, positions, inv_freq, yq, yk));
}

extern "C" int nott_qk_norm_rope_bwd(nott_ctx ctx, const nott_qk_rope_desc* d, nott_dtype dtype, const void* dyq,
                                     const void* dyk, const void* q, const void* k, const void* gamma_q,
                                     const void* gamma_k, const int64_t* positions, const double* inv_freq, void* dq,
                                     void* dk, float* dgamma_q, float* dgamma_k, int accumulate) {
    NOTT_CHECK_CTX(ctx);
    const int st = check(ctx, d, dtype, "nott_qk_norm_rope_bwd");
    if (st != NOTT_OK) return st;
    NOTT_REQUIRE(ctx, d->norm || (!gamma_q && !gamma_k && !dgamma_q && !dgamma_k),
                 "nott_qk_norm_rope_bwd: a weight needs the norm");
    nott::DeviceScope scope(ctx->device);
    if (d->b * d->t * (d->hq + d->hk) == 0) {
        // no token: the weights' gradients sum over nothing
        for (float* g : {dgamma_q, dgamma_k})
            if (g && !accumulate && nott_zero(ctx, (int64_t)sizeof(float) * d->dh, g) != NOTT_OK) return NOTT_ERR_HIP;
        return NOTT_OK;
    }
    NOTT_REQUIRE(ctx, (d->hq == 0 || (dyq && dq)) && (d->hk == 0 || (dyk && dk)), "nott_qk_norm_rope_bwd: null buffer");
    NOTT_REQUIRE(ctx, !d->norm || ((d->hq == 0 || q) && (d->hk == 0 || k)), "nott_qk_norm_rope_bwd: the norm needs q and k");
    NOTT_REQUIRE(ctx, d->rot == 0 || (positions && inv_freq), "nott_qk_norm_rope_bwd: null positions or inv_freq");
    if (dtype == NOTT_F32)
        return backward(ctx, make_args<float>(*d, q, k, dyq, dyk, gamma_q, gamma_k, positions, inv_freq, dq, dk), dgamma_q,
                        dgamma_k, accumulate);
    return backward(ctx, make_args<bf16_t>(*d, q, k, dyq, dyk, gamma_q, gamma_k, positions, inv_freq, dq, dk), dgamma_q,
                    dgamma_k, accumulate);
}
