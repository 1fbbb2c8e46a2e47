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
    int64_t items;      // tokens · (hq + hk)
    FastDiv by_heads, by_t, by_width;   // by_width: pairs of a token's table
    float* partial;     // backward: [grid][2·dh] sums of dz·x̂, q then k; null: not asked for
};

__device__ __forceinline__ int64_t at(const int64_t (&s)[3], uint32_t b, uint32_t t, uint32_t h) {
    return b * s[0] + t * s[1] + h * s[2];
}

// Any head size and alignment: a wave per head, element e = 64·v + lane.
// Every load of a head comes before its stores (the stores wait for the loaded
// values), so an output may be its input.
template <typename T, bool BWD>
__global__ __launch_bounds__(256) void rope_any_kernel(RopeArgs<T> a) {
    constexpr int V = kMaxHead / 64;
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    const int half = a.turns.half;
    float dgq[V], dgk[V];
#pragma unroll
    for (int v = 0; v < V; ++v) dgq[v] = dgk[v] = 0.f;
    for (int64_t item = (int64_t)blockIdx.x * 4 + wid; item < a.items; item += (int64_t)gridDim.x * 4) {
        uint32_t token, head, bi, ti;
        a.by_heads.divmod((uint32_t)item, token, head);
        a.by_t.divmod(token, bi, ti);
        const bool is_q = head < (uint32_t)a.q.n;
        const Heads<T>& h = is_q ? a.q : a.k;
        if (!is_q) head -= a.q.n;
        const T* x = h.x + at(h.xs, bi, ti, head);
        const T* dy = BWD ? h.dy + at(h.ys, bi, ti, head) : nullptr;
        T* out = BWD ? h.out + at(h.os, bi, ti, head) : h.out + at(h.ys, bi, ti, head);
        const bool has_x = !BWD || a.norm;
        float xv[V], ov[V];
        float ss = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int e = 64 * v + lane;
            xv[v] = has_x && e < a.dh ? Io<T>::ld(x, e) : 0.f;
            ss = fmaf(xv[v], xv[v], ss);
        }
        float r = 1.f;
        if (a.norm) r = rsqrtf(wave_sum(ss) / (float)a.dh + a.eps);
        float dot = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int e = 64 * v + lane;
            if (e >= a.dh) {
                ov[v] = 0.f;
                continue;
            }
            const float g = h.gamma ? Io<T>::ld(h.gamma, e) : 1.f;
            // the other element of e's pair (e itself past the rotated ones)
            const bool rotated = e < 2 * half;
            const bool second = a.turns.interleaved ? (e & 1) : e >= half;
            const int other = !rotated ? e : a.turns.interleaved ? e ^ 1 : second ? e - half : e + half;
            float c = 1.f, s = 0.f;
            if (rotated) a.turns.turn(token, a.turns.interleaved ? e >> 1 : second ? e - half : e, c, s);
            if constexpr (!BWD) {
                const float z = xv[v] * r * g;
                const float zo = Io<T>::ld(x, other) * r * (h.gamma ? Io<T>::ld(h.gamma, other) : 1.f);
                ov[v] = second ? fmaf(zo, s, z * c) : fmaf(-zo, s, z * c);
            } else {
                const float d = Io<T>::ld(dy, e), od = Io<T>::ld(dy, other);
                const float dz = second ? fmaf(-od, s, d * c) : fmaf(od, s, d * c);
                const float xh = xv[v] * r;
                if (is_q) dgq[v] = fmaf(dz, xh, dgq[v]);
                else dgk[v] = fmaf(dz, xh, dgk[v]);
                ov[v] = dz * g;
                dot = fmaf(ov[v], xh, dot);
            }
        }
        if constexpr (BWD) {
            if (a.norm) {
                dot = wave_sum(dot) / (float)a.dh;
#pragma unroll
                for (int v = 0; v < V; ++v) ov[v] = r * (ov[v] - xv[v] * r * dot);
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int e = 64 * v + lane;
            if (e < a.dh) Io<T>::st(out, e, ov[v]);
        }
    }
    if constexpr (BWD) {
        if (!a.partial) return;
        __shared__ float red[2][kMaxHead];
        for (int w = 0; w < 4; ++w) {
            if (wid == w) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    red[0][64 * v + lane] = w ? red[0][64 * v + lane] + dgq[v] : dgq[v];
                    red[1][64 * v + lane] = w ? red[1][64 * v + lane] + dgk[v] : dgk[v];
                }
            }
            __syncthreads();
        }
        float* p = a.partial + (int64_t)blockIdx.x * 2 * a.dh;
        for (int e = threadIdx.x; e < a.dh; e += 256) {
            p[e] = red[0][e];
            p[a.dh + e] = red[1][e];
        }
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
                auto turn2 = [](float& a, float& b, float c, float s) {
                    if (BWD) s = -s;
                    const float y = fmaf(-b, s, a * c);
                    b = fmaf(a, s, b * c);
                    a = y;
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
                        turn2(p[e], p[e + 1], cs.x, cs.y);
                        turn2(p[e + 2], p[e + 3], cs.z, cs.w);
                        turn2(q[e], q[e + 1], ct.x, ct.y);
                        turn2(q[e + 2], q[e + 3], ct.z, ct.w);
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
    a.items = d.b * d.t * (d.hq + d.hk);
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
Launch plan(nott_ctx ctx, const RopeArgs<T>& a, bool bwd) {
    constexpr int E = Pack16<T>::N, kGroups = sizeof(T) == 2 ? 3 : 4;
    Launch l{};
    const int slots = (a.dh / E + 1) / 2, pairs = table_pairs(a);
    for (l.lph = 2; l.lph < slots;) l.lph *= 2;
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

template <typename T>
int forward(nott_ctx ctx, const RopeArgs<T>& a) {
    if (in_chunks(a, false)) {
        launch_vec<T, false>(ctx, plan(ctx, a, false), a);
    } else {
        const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(a.items, 4), 32 * (int64_t)ctx->num_cu);
        hipLaunchKernelGGL((rope_any_kernel<T, false>), dim3(grid), dim3(256), 0, ctx->stream, a);
    }
    return nott::launch_status(ctx, "qk_norm_rope");
}

template <typename T>
int backward(nott_ctx ctx, RopeArgs<T> a, float* dgq, float* dgk, int accumulate) {
    const bool vec = in_chunks(a, true);
    Launch l = vec ? plan(ctx, a, true) : Launch{};
    if (!vec) l.grid = (unsigned)std::min<int64_t>(ceil_div(a.items, 4), 8 * (int64_t)ctx->num_cu);
    if (a.norm && (dgq || dgk)) {
        a.partial = static_cast<float*>(nott::workspace(ctx, sizeof(float) * 2 * (size_t)a.dh * l.grid));
        if (!a.partial) return NOTT_ERR_ALLOC;
    }
    if (vec) launch_vec<T, true>(ctx, l, a);
    else hipLaunchKernelGGL((rope_any_kernel<T, true>), dim3(l.grid), dim3(256), 0, ctx->stream, a);
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
