// Log probabilities of given tokens, with the entropy of each row and its most
// likely tokens, and their gradient.  Per row of logits, z = scale·logit:
//   m = max z, S = Σ exp(z − m), T = Σ exp(z − m)·(z − m)
//   lse = m + log S, logprob = (z_y − m) − log S, entropy = log S − T/S
//   dlogit_j = scale·(dlp·([j = y] − p_j) − dH·p_j·(log p_j + H)), p = exp(z − lse)
// Forward: one read of the row.  m, S and T are carried together: with a new
// maximum m' and a = exp(m − m'), S' = a·S and T' = a·(T + S·(m − m')).  The same
// running maxima give the top tokens: the top-th largest of 64 maxima over 64
// disjoint shares of the row is a bound that at least `top` elements reach and
// few more do (24 of any number for 20); what the few threads whose own maximum
// reaches it have read is read again, by all threads together.
// Backward: one read and one write.
#include "common.hpp"

namespace {

using nott::ceil_div;

constexpr int64_t kIgnoreIndex = -100;
constexpr int kMaxTop = 64;
constexpr int kUnroll = 4;          // 16-byte groups in flight per thread
constexpr int kMaxSplits = 64;      // a merging wave has a lane for each
constexpr float kLn2 = 0.69314718f;
// Logits of −inf or the type's lowest value mask a token: below this (times scale)
// there is nothing.  As the maximum's first value it keeps −inf − (−inf) out.
constexpr float kNothing = -1e30f;
// Exponents (base 2) are not taken below this: 0·(−inf) is no part of a sum.
constexpr float kLeast = -300.f;

// z = scale·logit; to_log2 = scale·log2 e; first: the maximum of no live logit.
struct Scale {
    float scale, to_log2, first;
};

// The running statistics of a part of a row: the largest logit m, s = Σ 2^w and
// t = Σ w·2^w with w = (logit − m)·to_log2.  A NaN stays in s.
struct Stats {
    float m, s, t;
    // Carries s and t over to the maximum n >= m.
    __device__ __forceinline__ void raise(float n, const Scale& sc) {
        const float d = fmaxf((m - n) * sc.to_log2, kLeast);
        const float a = __builtin_amdgcn_exp2f(d);
        t = a * fmaf(s, d, t);
        s *= a;
        m = n;
    }
    template <int N>
    __device__ __forceinline__ void add(const float (&v)[N], const Scale& sc) {
        float n = m;
#pragma unroll
        for (int e = 0; e < N; ++e) n = fmaxf(n, v[e]);
        raise(n, sc);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            // the difference first: n·to_log2 rounded would leave 2^-24 of |n| in every
            // exponent (rows masked with −1e9, logits with a common offset)
            const float w = (v[e] - n) * sc.to_log2;
            const float p = __builtin_amdgcn_exp2f(w);
            s += p;
            t = fmaf(p, fmaxf(w, kLeast), t);
        }
    }
    __device__ __forceinline__ void merge(Stats o, const Scale& sc) {
        const float n = fmaxf(m, o.m);
        raise(n, sc);
        o.raise(n, sc);
        s += o.s;
        t += o.t;
    }
    __device__ __forceinline__ void merge_wave(const Scale& sc) {
#pragma unroll
        for (int i = 1; i < 64; i <<= 1) merge(Stats{__shfl_xor(m, i), __shfl_xor(s, i), __shfl_xor(t, i)}, sc);
    }
};

// Order of the most likely tokens as one whole number: the value in an order that
// integers keep (−0 as +0, NaN above all), then the lower column.  0 and all ones
// are no keys.
__device__ __forceinline__ uint64_t top_key(float z, uint32_t col) {
    uint32_t u = __builtin_bit_cast(uint32_t, z + 0.f);
    u = z != z ? 0xfffffffeu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
    return ((uint64_t)u << 32) | (uint32_t)~col;
}

template <int CTRL>
__device__ __forceinline__ uint64_t dpp_max64(uint64_t v) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, 0xf, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, 0xf, 0xf, false);
    return max(v, ((uint64_t)hi << 32) | lo);
}
template <int L>
__device__ __forceinline__ uint64_t lane_u64(uint64_t v) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, L), hi = __builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), L);
    return ((uint64_t)hi << 32) | lo;
}
// The largest of the wave's keys, as wave_max (a shuffled one takes 0.4 us).
__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
    v = dpp_max64<0xB1>(v);
    v = dpp_max64<0x4E>(v);
    v = dpp_max64<0x141>(v);
    v = dpp_max64<0x140>(v);
    return max(max(lane_u64<0>(v), lane_u64<16>(v)), max(lane_u64<32>(v), lane_u64<48>(v)));
}

// The top-th largest of the wave's 64 values (none a NaN): up to 16 by taking the
// largest away one after the other, past that by every lane's rank.
__device__ __forceinline__ float wave_nth(float v, int top) {
    const int lane = (int)threadIdx.x & 63;
    if (top <= 16) {
        float m = wave_max(v);
        for (int i = 1; i < top; ++i) {
            const uint64_t hit = __ballot(v == m);
            if (lane == __ffsll((unsigned long long)hit) - 1) v = -INFINITY;
            m = wave_max(v);
        }
        return m;
    }
    int rank = 0;
#pragma unroll
    for (int j = 0; j < 64; ++j) {
        const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), j));
        rank += w > v || (w == v && j < lane) ? 1 : 0;
    }
    const uint64_t hit = __ballot(rank == top - 1);
    return __shfl(v, __ffsll((unsigned long long)hit) - 1);
}

struct FwdOut {
    float* logprob;
    float* entropy;
    float* lse;
    float* top_logprob;
    int64_t* top_index;
    unsigned long long* err;
};

// log p of a logit in a row of statistics st, logs = log st.s.
__device__ __forceinline__ float log_p(float x, const Stats& st, float logs, const Scale& sc) {
    return st.s == 0.f || x * sc.scale < kNothing ? -INFINITY : (x - st.m) * sc.scale - logs;
}

// The row's outputs from its statistics.
template <typename T>
__device__ __forceinline__ void write_row(const FwdOut& o, int64_t row, int64_t y, int64_t c, const T* z, const Scale& sc,
                                          const Stats& st, float logs) {
    const bool empty = st.s == 0.f;   // every token masked
    float lp = 0.f;
    if (y >= 0 && y < c) lp = log_p(Io<T>::ld(z, y), st, logs, sc);
    else if (y != kIgnoreIndex) atomicAdd(o.err, 1ull);
    o.logprob[row] = lp;
    if (o.lse) o.lse[row] = empty ? -INFINITY : fmaf(st.m, sc.scale, logs);
    if (o.entropy) o.entropy[row] = empty ? 0.f : logs - st.t * kLn2 / st.s;
}

template <typename T>
__device__ __forceinline__ void write_top(const FwdOut& o, int64_t at, uint64_t key, const T* z, const Stats& st,
                                          float logs, const Scale& sc) {
    const uint32_t col = ~(uint32_t)key;
    o.top_index[at] = col;
    o.top_logprob[at] = log_p(Io<T>::ld(z, col), st, logs, sc);
}

template <typename T>
__device__ __forceinline__ typename Pack16<T>::Raw minus_inf() {
    if constexpr (sizeof(T) == 2) return u32x4{0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u};
    else return f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
}

// A part of a row of any alignment as its whole 16-byte groups (group i at base +
// i·G) and the fewer than 2·G elements before and after them, one per thread.
template <typename T>
struct Span {
    static constexpr int G = Pack16<T>::N;
    const T* base;
    int groups;
    int single;   // this thread's single element from p, −1: none
    __device__ __forceinline__ Span(const T* p, int len) {
        const int s0 = min((int)((G - ((uintptr_t)p / sizeof(T)) % G) % G), len);
        groups = (len - s0) / G;
        base = p + s0;
        const int tail = s0 + groups * G, tid = (int)threadIdx.x;
        single = tid < s0 ? tid : tail + (tid - s0) < len ? tail + (tid - s0) : -1;
    }
};

// A workgroup per row, or with splits > 1 per part of `chunk` columns, whose
// statistics and top keys go to `stats` [row][split] and `keys` [row][split][top].
// LDS holds `cap` candidates for the top tokens; a row in which more reach the
// bound is scanned for each: many equal logits, too few live ones for a bound (fewer
// than `top` of the 64 shares hold one), and of the one-wave rows (cap 256) with top
// past about 60 ordinary ones too (the bound is then about the least of 64 maxima,
// which 64·H(64) = 304 elements reach in the mean).
// Bound by memory (one read of the logits), then by the exponential and seven more
// instructions an element.
// 16384x32000 bf16, top 5, 188 us (5.6 TB/s; 245 in the mean of twenty in a row);
// 8x128256 bf16, top 8, in parts of 4096 columns and more 7.1 us and 4.6 to join them.
template <typename T, int NT>
__global__ __launch_bounds__(NT) void logprob_kernel(const T* __restrict__ logits, const int64_t* __restrict__ labels,
                                                     int64_t c, int chunk, Scale sc, int top, int cap, FwdOut o,
                                                     Stats* __restrict__ stats, uint64_t* __restrict__ keys) {
    constexpr int G = Pack16<T>::N, W = NT / 64;
    extern __shared__ uint64_t cand[];
    __shared__ Stats part[W];
    __shared__ float share[NT];
    __shared__ float bound_s;
    __shared__ int count, hot_count;
    __shared__ int hot[NT];
    __shared__ uint64_t red[W];
    const int tid = (int)threadIdx.x, lane = tid & 63, wid = tid >> 6;
    const int64_t row = blockIdx.x;
    const T* z = logits + row * c;
    const int64_t j0 = (int64_t)blockIdx.y * chunk;
    const int len = (int)min((int64_t)chunk, c - j0);
    const Span<T> sp(z + j0, len);
    Stats st{sc.first, 0.f, 0.f};
    const int full = sp.groups / (NT * kUnroll);
    for (int i = 0; i < full; ++i) {
        typename Pack16<T>::Raw raw[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            raw[u] = Pack16<T>::template raw<true>(sp.base + (int64_t)((i * kUnroll + u) * NT + tid) * G);
        float v[kUnroll * G];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) Pack16<T>::unpack(raw[u], reinterpret_cast<float(&)[G]>(v[u * G]));
        st.add(v, sc);
    }
    if (full * kUnroll * NT < sp.groups) {   // the rest, its loads in flight together
        const int k = full * kUnroll * NT + tid;
        typename Pack16<T>::Raw raw[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            raw[u] = Pack16<T>::template raw<true>(sp.base + (int64_t)min(k + u * NT, sp.groups - 1) * G);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            if (full * kUnroll * NT + u * NT >= sp.groups) break;
            float v[G];
            Pack16<T>::unpack(k + u * NT < sp.groups ? raw[u] : minus_inf<T>(), v);
            st.add(v, sc);
        }
    }
    if (sp.single >= 0) {
        const float v[1] = {Io<T>::ld(z + j0, sp.single)};
        st.add(v, sc);
    }
    const float own = st.s != st.s ? INFINITY : st.m;   // a NaN is among the largest
    if (tid == 0) count = hot_count = 0;
    share[tid] = own;
    st.merge_wave(sc);
    if (lane == 0) part[wid] = st;
    __syncthreads();
    st = part[0];
#pragma unroll
    for (int i = 1; i < W; ++i) st.merge(part[i], sc);
    const float logs = logf(st.s);
    const bool whole = gridDim.y == 1;
    const int64_t at = row * gridDim.y + blockIdx.y;
    if (tid == 0) {
        if (whole) write_row(o, row, labels[row], c, z, sc, st, logs);
        else stats[at] = st;
    }
    if (top == 0) return;
    if (wid == 0) {
        float v = share[lane];
#pragma unroll
        for (int i = 1; i < W; ++i) v = fmaxf(v, share[i * 64 + lane]);
        v = wave_nth(v, top);
        if (lane == 0) bound_s = v;
    }
    __syncthreads();
    // no bound among live logits: every element is a candidate
    const float bound = bound_s > sc.first ? bound_s : -INFINITY;
    auto offer = [&](float x, int64_t col) {
        if (x < bound) return;
        const int i = atomicAdd(&count, 1);
        if (i < cap) cand[i] = top_key(x, (uint32_t)col);
    };
    if (!(own < bound)) {
        hot[atomicAdd(&hot_count, 1)] = tid;
        if (sp.single >= 0) offer(Io<T>::ld(z + j0, sp.single), j0 + sp.single);
    }
    __syncthreads();
    // groups tid, tid + NT, ... of the hot threads
    const int64_t first = j0 + (sp.base - (z + j0));
    const int nh = hot_count, all = nh * ((sp.groups + NT - 1) / NT);
    for (int i = tid; i < all; i += NT * 2) {
        int k[2];
        typename Pack16<T>::Raw raw[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int w = min(i + u * NT, all - 1), turn = w / nh;
            k[u] = hot[w - turn * nh] + turn * NT;
            raw[u] = Pack16<T>::template raw<false>(sp.base + (int64_t)min(k[u], sp.groups - 1) * G);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if (i + u * NT >= all || k[u] >= sp.groups) continue;
            float v[G];
            Pack16<T>::unpack(raw[u], v);
#pragma unroll
            for (int e = 0; e < G; ++e) offer(v[e], first + (int64_t)k[u] * G + e);
        }
    }
    __syncthreads();
    const int n = count;
    auto put = [&](int i, uint64_t key) {
        if (whole) write_top(o, row * top + i, key, z, st, logs, sc);
        else keys[at * top + i] = key;
    };
    if (n <= cap) {
        for (int i = tid; i < n; i += NT) {
            const uint64_t key = cand[i];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += cand[j] > key ? 1 : 0;
            if (rank < top) put(rank, key);
        }
        for (int i = n + tid; i < top; i += NT) put(i, 0);   // only in a part shorter than top
        return;
    }
    uint64_t last = ~uint64_t(0);
    for (int i = 0; i < top; ++i) {
        uint64_t best = 0;
        for (int j = tid; j < len; j += NT) {
            const uint64_t key = top_key(Io<T>::ld(z + j0, j), (uint32_t)(j0 + j));
            if (key < last && key > best) best = key;
        }
        best = wave_max64(best);
        if (lane == 0) red[wid] = best;
        __syncthreads();
        last = red[0];
#pragma unroll
        for (int w = 1; w < W; ++w) last = max(last, red[w]);
        __syncthreads();
        if (tid == 0) put(i, last);
    }
}

// The rows from their parts, a wave each: lane s has split s's statistics and its
// sorted keys, of which the largest head is taken `top` times.
template <typename T>
__global__ __launch_bounds__(64) void logprob_merge_kernel(const T* __restrict__ logits,
                                                           const int64_t* __restrict__ labels, int64_t c, int splits,
                                                           Scale sc, int top, FwdOut o, const Stats* __restrict__ stats,
                                                           const uint64_t* __restrict__ keys) {
    const int lane = (int)threadIdx.x;
    const int64_t row = blockIdx.x;
    const bool mine = lane < splits;
    const uint64_t* list = keys + (row * splits + lane) * top;
    Stats st = mine ? stats[row * splits + lane] : Stats{sc.first, 0.f, 0.f};
    int taken = 0;
    uint64_t head = mine && top ? list[0] : 0;
    st.merge_wave(sc);
    const float logs = logf(st.s);
    const T* z = logits + row * c;
    if (lane == 0) write_row(o, row, labels[row], c, z, sc, st, logs);
    uint64_t won = 0;   // lane i: the i-th
    for (int i = 0; i < top; ++i) {
        const uint64_t best = wave_max64(head);
        if (lane == i) won = best;
        if (head == best) {
            ++taken;
            head = taken < top ? list[taken] : 0;
        }
    }
    if (lane < top) write_top(o, row * top + lane, won, z, st, logs, sc);
}

// The gradient of one part of a row: NT·kUnroll groups, part 0 with the single
// elements.  A group's loads are all issued before its stores, so dlogits may be
// logits.  Bound by memory: 4096x50257 fp32 with entropies 284 us (5.8 TB/s).
template <typename T, int NT>
__global__ __launch_bounds__(NT) void logprob_bwd_kernel(const T* logits, const int64_t* __restrict__ labels, int64_t c,
                                                         uint32_t parts, FastDiv by_parts, float scale,
                                                         const float* __restrict__ lse,
                                                         const float* __restrict__ entropy,
                                                         const float* __restrict__ dlogprob,
                                                         const float* __restrict__ dentropy, T* dlogits) {
    constexpr int G = Pack16<T>::N;
    uint32_t r32, part;
    by_parts.divmod(blockIdx.x, r32, part);
    const int64_t row = r32;
    const int tid = (int)threadIdx.x;
    const T* z = logits + row * c;
    T* dz = dlogits + row * c;
    const Span<T> sp(z, (int)c);
    const int k0 = (int)part * NT * kUnroll + tid;
    typename Pack16<T>::Raw raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) raw[u] = minus_inf<T>();
    if (sp.groups > 0) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            raw[u] = Pack16<T>::template raw<true>(sp.base + (int64_t)min(k0 + u * NT, sp.groups - 1) * G);
    }
    const int64_t y = labels[row];
    const bool given = y >= 0 && y < c;
    const float l = lse[row], h = dentropy ? entropy[row] : 0.f;
    const float dl = given ? dlogprob[row] : 0.f, dh = dentropy ? dentropy[row] : 0.f;
    const int first = (int)(sp.base - z);
    auto grad = [&](float x, int col) {
        const float lp = fmaf(x, scale, -l);
        // below −200 (masked logits: −inf and the type's lowest value) p is 0
        float g = -exp_fine(lp < -200.f ? -200.f : lp) * fmaf(dh, fmaxf(lp, -200.f) + h, dl);
        if (col == (int)y) g += dl;
        return l == -INFINITY ? 0.f : g * scale;
    };
    const bool vec = ((uintptr_t)(dz + first) % 16) == 0;
    const float xs = part == 0 && sp.single >= 0 ? Io<T>::ld(z, sp.single) : 0.f;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int k = k0 + u * NT;
        if (k >= sp.groups) break;
        const int col = first + k * G;
        float v[G];
        Pack16<T>::unpack(raw[u], v);
#pragma unroll
        for (int e = 0; e < G; ++e) v[e] = grad(v[e], col + e);
        if (vec) {
            Pack16<T>::template st<true>(dz + col, v);
        } else {
#pragma unroll
            for (int e = 0; e < G; ++e) Io<T>::st(dz, col + e, v[e]);
        }
    }
    if (part == 0 && sp.single >= 0) Io<T>::st(dz, sp.single, grad(xs, sp.single));
}

// Workgroups of a launch: its threads are counted in 32 bits.
constexpr int64_t kMaxGrid = int64_t(1) << 23;
// Threads of a row: one wave up to 2048 columns, and up to 4096 where there are rows
// for every SIMD.
int row_threads(nott_ctx ctx, int64_t n, int64_t c) {
    return c <= 2048 || (c <= 4096 && n >= 8 * (int64_t)ctx->num_cu) ? 64 : 256;
}

template <typename T>
int forward(nott_ctx ctx, int64_t n, int64_t c, const T* logits, const int64_t* labels, double scale, int top,
            const FwdOut& o) {
    const Scale sc{(float)scale, (float)(scale * 1.4426950408889634), (float)std::max(-1e30 / scale, -3e38)};
    const int nt = row_threads(ctx, n, c);
    // Fewer rows than fill the card are split, into parts of at least 4096 columns.
    int64_t splits = 1;
    if (n < 4 * ctx->num_cu)
        splits = std::max<int64_t>(1, std::min<int64_t>({kMaxSplits, 4 * (int64_t)ctx->num_cu / n, c / 4096}));
    int64_t chunk = splits == 1 ? c : ceil_div(ceil_div(c, splits), 64) * 64;
    splits = ceil_div(c, chunk);
    Stats* stats = nullptr;
    uint64_t* keys = nullptr;
    if (splits > 1) {
        const size_t sb = (sizeof(Stats) * (size_t)(n * splits) + 255) & ~size_t(255);
        char* ws = static_cast<char*>(nott::optional_workspace(ctx, sb + sizeof(uint64_t) * (size_t)(n * splits * top)));
        stats = reinterpret_cast<Stats*>(ws);
        keys = reinterpret_cast<uint64_t*>(ws + sb);
        if (!ws) splits = 1, chunk = c;
    }
    const int cap = top == 0 ? 0 : nt == 64 ? 256 : 1024;
    for (int64_t r = 0; r < n; r += kMaxGrid) {   // more than one only for rows that are not split
        const dim3 grid((unsigned)std::min(kMaxGrid, n - r), (unsigned)splits);
        const FwdOut at{o.logprob + r, o.entropy ? o.entropy + r : nullptr, o.lse ? o.lse + r : nullptr,
                        top ? o.top_logprob + r * top : nullptr, top ? o.top_index + r * top : nullptr, o.err};
        auto launch = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, grid, dim3(nt), sizeof(uint64_t) * cap, ctx->stream, logits + r * c, labels + r, c,
                               (int)chunk, sc, top, cap, at, stats, keys);
        };
        if (nt == 64) launch(logprob_kernel<T, 64>);
        else launch(logprob_kernel<T, 256>);
    }
    if (splits > 1)
        hipLaunchKernelGGL(logprob_merge_kernel<T>, dim3((unsigned)n), dim3(64), 0, ctx->stream, logits, labels, c,
                           (int)splits, sc, top, o, stats, keys);
    return nott::launch_status(ctx, "token_logprob");
}

template <typename T>
int backward(nott_ctx ctx, int64_t n, int64_t c, const T* logits, const int64_t* labels, float scale, const float* lse,
             const float* entropy, const float* dlogprob, const float* dentropy, T* dlogits) {
    const int nt = c <= 2048 ? 64 : 256;
    const int64_t parts = std::max<int64_t>(1, ceil_div(c, (int64_t)nt * kUnroll * Pack16<T>::N));
    const int64_t rows = std::max<int64_t>(1, kMaxGrid / parts);
    for (int64_t r = 0; r < n; r += rows) {
        const unsigned grid = (unsigned)(std::min(rows, n - r) * parts);
        const FastDiv by((uint32_t)parts);
        auto launch = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(grid), dim3(nt), 0, ctx->stream, logits + r * c, labels + r, c, (uint32_t)parts,
                               by, scale, lse + r, entropy ? entropy + r : nullptr, dlogprob + r,
                               dentropy ? dentropy + r : nullptr, dlogits + r * c);
        };
        if (nt == 64) launch(logprob_bwd_kernel<T, 64>);
        else launch(logprob_bwd_kernel<T, 256>);
    }
    return nott::launch_status(ctx, "token_logprob backward");
}

// What fp32 holds, with room for a logit's product (a scale that rounds to 0 would make
// NaN of a masked token).
bool valid_scale(double scale) { return scale >= 1e-30 && scale < 1e30; }

}  // namespace

extern "C" int nott_token_logprob_fwd(nott_ctx ctx, nott_dtype dtype, int64_t n, int64_t c, const void* logits,
                                      const int64_t* labels, double scale, int64_t top, float* logprob, float* entropy,
                                      float* lse, float* top_logprob, int64_t* top_index) {
    NOTT_CHECK_CTX(ctx);
    NOTT_REQUIRE(ctx, nott::valid_dtype(dtype), "nott_token_logprob_fwd: bad dtype");
    NOTT_REQUIRE(ctx, n >= 0 && c > 0 && n < (int64_t(1) << 31) && c < (int64_t(1) << 31),
                 "nott_token_logprob_fwd: need 0 <= n and 0 < c, both below 2^31");
    NOTT_REQUIRE(ctx, valid_scale(scale), "nott_token_logprob_fwd: scale must be 1e-30 to 1e30");
    NOTT_REQUIRE(ctx, top >= 0 && top <= kMaxTop && top <= c, "nott_token_logprob_fwd: top must be 0 to min(c, 64)");
    if (n == 0) return NOTT_OK;
    NOTT_REQUIRE(ctx, logits && labels && logprob, "nott_token_logprob_fwd: null buffer");
    NOTT_REQUIRE(ctx, top == 0 || (top_logprob && top_index), "nott_token_logprob_fwd: top needs top_logprob and top_index");
    nott::DeviceScope scope(ctx->device);
    const FwdOut o{logprob, entropy, lse, top_logprob, top_index, ctx->err_word};
    if (dtype == NOTT_F32) return forward(ctx, n, c, static_cast<const float*>(logits), labels, scale, (int)top, o);
    return forward(ctx, n, c, static_cast<const bf16_t*>(logits), labels, scale, (int)top, o);
}

extern "C" int nott_token_logprob_bwd(nott_ctx ctx, nott_dtype dtype, int64_t n, int64_t c, const void* logits,
                                      const int64_t* labels, double scale, const float* lse, const float* entropy,
                                      const float* dlogprob, const float* dentropy, void* dlogits) {
    NOTT_CHECK_CTX(ctx);
    NOTT_REQUIRE(ctx, nott::valid_dtype(dtype), "nott_token_logprob_bwd: bad dtype");
    NOTT_REQUIRE(ctx, n >= 0 && c > 0 && n < (int64_t(1) << 31) && c < (int64_t(1) << 31),
                 "nott_token_logprob_bwd: need 0 <= n and 0 < c, both below 2^31");
    NOTT_REQUIRE(ctx, valid_scale(scale), "nott_token_logprob_bwd: scale must be 1e-30 to 1e30");
    if (n == 0) return NOTT_OK;
    NOTT_REQUIRE(ctx, logits && labels && lse && dlogprob && dlogits, "nott_token_logprob_bwd: null buffer");
    NOTT_REQUIRE(ctx, !dentropy || entropy, "nott_token_logprob_bwd: dentropy needs entropy");
    nott::DeviceScope scope(ctx->device);
    if (dtype == NOTT_F32)
        return backward(ctx, n, c, static_cast<const float*>(logits), labels, (float)scale, lse, entropy, dlogprob,
                        dentropy, static_cast<float*>(dlogits));
    return backward(ctx, n, c, static_cast<const bf16_t*>(logits), labels, (float)scale, lse, entropy, dlogprob, dentropy,
                    static_cast<bf16_t*>(dlogits));
}
