// Differential attention: two softmax maps a head, the second subtracted with a learned
// weight (flash-style, MFMA), forward and backward.
//
//   z_r = q_r·k_rᵀ·scale, p_r = softmax(z_r) for r = 1, 2;  o_r = p_r·v;  o = o_1 − λ·o_2
// backward, from the forward's o, o_2 and log-sum-exps:
//   dp = dO·vᵀ (one product for both maps),  D_2 = dO·o_2,  D_1 = dO·o + λ·D_2
//   dz_1 = p_1∘(dp − D_1),  dz_2 = −λ·p_2∘(dp − D_2)
//   dq_r = dz_r·k_r·scale,  dk_r = dz_rᵀ·q_r·scale,  dv = (p_1 − λ·p_2)ᵀ·dO,  dλ = −D_2
// So a pair of query and key costs 4·dh + 4·dv operations forward and, with two passes
// that both form the scores and dp, 16·dh + 6·dv backward (20·dh + 6·dv where dk and dv are
// apart, a third pass); v and dO are read, and dp and dv formed, once for both maps.
//
// Rows.  All queries of the heads that share a key head are one list of rows, query by
// query (row = query·group + head of the group), so a workgroup's rows share the tiles of
// keys and values however many heads there are, and dk and dv are summed over the group in
// the accumulator.  What a row sees is one number, its visible keys: keys below it.
//
// bf16 with 16-byte aligned rows runs on 32×32×16 MFMAs (namespace mx), in the layouts of
// attention.hip's kernels: scores are formed transposed, so that a lane owns a row.
// fp32, and rows that are not aligned, take the 16×16 kernels (namespace any).
// Probabilities (forward), p_1 − λ·p_2 and dz enter the second products as a bf16 value and
// the bf16 value of its remainder, off by 2^-16: o_1 and λ·o_2 nearly cancel where the maps
// resemble each other, and what one rounding (2^-8) leaves of each does not.  So the results
// are off by their own rounding (relative error against 64 bits 1.7e-3, the least for bf16;
// with one rounding 2.0e-3 to 2.4e-3, and up to 10 times the tolerance of tests of such
// maps).  The second half of the products costs 8 x 1024 tokens of 8 heads of 64 + 128
// columns 47 -> 58 us forward and 162 -> 171 backward, 4096 tokens of 16 heads on 4 of
// 128 + 256 1396 -> 1550 backward, a step against a cache nothing.  (Times of other choices
// beside the kernels were taken with one rounding.)
// Few rows against many keys (a decoding step): the keys are split over workgroups and
// waves, and a second kernel joins the parts.
// No atomics: every result is formed in a fixed order.
#include "attention_tile.hpp"
#include "lds_dma.hpp"

#include <atomic>
#include <type_traits>

namespace {

using namespace nott::attn;
using nott::ceil_div;
using nott::launch_status;

constexpr int64_t kMostBlocks = 1 << 22;    // of 256 threads, in a launch (its threads fit 32 bits)
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Params {
    int32_t t, s, dh, dv, h, hk, group, rows;   // rows = t·group, of a key head
    int32_t causal, token_lam, vec, nsplit;
    int32_t near;         // 128 rows of q, k, v, dO lie within 2^31 bytes: 32-bit offsets reach a tile's
    float scale;
    FastDiv by_group;
    int64_t q[3], k[3], v[3], o[3], od[3], dq[3], dk[3], dv_[3];   // strides: batch, token, head (od: dO)
    const int32_t* lengths;
    const int32_t* start;
    const float* lam;
};

// One (batch, key head) pair and what its rows see.
struct Pair {
    int b, j, len, start;
    __device__ __forceinline__ Pair(const Params& p, int bk) {
        b = bk / p.hk;
        j = bk - b * p.hk;
        len = p.lengths ? max(0, min(p.s, p.lengths[b])) : p.s;
        start = p.start ? p.start[b] : 0;
    }
    // Keys that query i sees: those below this number.
    __device__ __forceinline__ int visible(const Params& p, int i) const {
        if (!p.causal) return len;
        return (int)max<int64_t>(0, min<int64_t>(len, (int64_t)start + i + 1));
    }
    // The first row that sees key k (p.rows or more: none).
    __device__ __forceinline__ int first_row(const Params& p, int k) const {
        if (!p.causal) return 0;
        return (int)min<int64_t>(p.rows, max<int64_t>(0, (int64_t)k - start) * p.group);
    }
};
struct RowAt {
    int i, head;
    __device__ __forceinline__ RowAt(const Params& p, const Pair& w, int row) {
        uint32_t qi, g;
        p.by_group.divmod((uint32_t)row, qi, g);
        i = (int)qi;
        head = w.j * p.group + (int)g;
    }
};
template <typename T>
__device__ __forceinline__ T* at(T* base, const int64_t (&st)[3], int b, int i, int head) {
    return base + (int64_t)b * st[0] + (int64_t)i * st[1] + (int64_t)head * st[2];
}
__device__ __forceinline__ float lambda_of(const Params& p, int b, const RowAt& r) {
    return p.lam[p.token_lam ? ((int64_t)b * p.t + r.i) * p.h + r.head : r.head];
}
__device__ __forceinline__ float* lse_at(const Params& p, float* lse, int b, const RowAt& r, int map) {
    return lse + ((int64_t)b * 2 * p.h + 2 * r.head + map) * p.t + r.i;
}
// Of a row's sum l: 0 where it sees no key; NaN (of a NaN score) stays NaN.
__device__ __forceinline__ float log_sum(float m, float l) { return l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2; }
__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }

// Rows' statistics that the dq pass hands to the dk/dv pass, [kStats][b·hk][rows]:
// log2(e)·lse of both maps, D_1, D_2, λ.
constexpr int kStats = 5;

// Partial results of split keys: acc [nsplit][b·hk][rows][2][dv], then {m, l}
// [nsplit][b·hk][rows][2] (m in log2; not divided by l).
struct Parts {
    float* acc;
    float* ml;
};

// Joins the parts (at most 64): a workgroup of WAVES waves a row.  Lane z weighs part z; a
// wave sums every WAVES-th part, its loads in flight beside those of the weights, and the
// waves' sums are added in order (a wave a row, a part after the other, took 17.7 us for
// 128 rows in 8 parts; four waves 4.8).  Up to 4 parts are one wave's loads
// (14000 rows in 3 parts 40.7 us with four waves, 15.9 with one).
constexpr int kMostParts = 64;
template <typename T, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void diff_join_kernel(Parts parts, T* __restrict__ o, T* __restrict__ o2,
                                                        float* __restrict__ lse, int64_t total, Params p) {
    __shared__ float sum[WAVES][2][256];
    const int64_t at_row = blockIdx.x;      // (b·hk + j)·rows + row
    const int wid = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int bk = (int)(at_row / p.rows), row = (int)(at_row - (int64_t)bk * p.rows);
    const float* ml = parts.ml + at_row * 4;
    const f32x4 mine = lane < p.nsplit ? *reinterpret_cast<const f32x4*>(ml + lane * total * 4)    // {m, l} of both maps
                                       : f32x4{-INFINITY, 0.f, -INFINITY, 0.f};
    constexpr int U = 4;        // parts of a wave at a time
    float a[U][2][4];
    auto load = [&](int z0) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int z = min(z0 + WAVES * u, p.nsplit - 1), d = lane + 64 * c;
                    a[u][k][c] = d < p.dv ? parts.acc[((z * total + at_row) * 2 + k) * p.dv + d] : 0.f;
                }
    };
    load(wid);
    const Pair w(p, bk);
    const RowAt r(p, w, row);
    const float lam = lambda_of(p, w.b, r);
    const float m[2] = {wave_max(mine.x), wave_max(mine.z)};
    const float f[2] = {mine.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mine.x - m[0]),
                        mine.z == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mine.z - m[1])};
    const float l[2] = {wave_sum(f[0] * mine.y), wave_sum(f[1] * mine.w)};
    float acc[2][4] = {};
    for (int z0 = wid; z0 < p.nsplit; z0 += WAVES * U) {
        if (z0 != wid) load(z0);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float fz = __shfl(f[k], min(z0 + WAVES * u, 63), 64);
                if (z0 + WAVES * u >= p.nsplit || fz == 0.f) continue;
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[k][c] = fmaf(fz, a[u][k][c], acc[k][c]);
            }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int c = 0; c < 4; ++c) sum[wid][k][lane + 64 * c] = acc[k][c];
    __syncthreads();
    const float i1 = inverse(l[0]), i2 = inverse(l[1]);
    for (int d = threadIdx.x; d < p.dv; d += 64 * WAVES) {
        float of[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            of[k] = sum[0][k][d];
#pragma unroll
            for (int w2 = 1; w2 < WAVES; ++w2) of[k] += sum[w2][k][d];
        }
        const float second = of[1] * i2;
        Io<T>::st(at(o, p.o, w.b, r.i, r.head), d, of[0] * i1 - lam * second);
        if (o2) Io<T>::st(o2, (((int64_t)w.b * p.t + r.i) * p.h + r.head) * p.dv + d, second);
    }
    if (threadIdx.x < 2) *lse_at(p, lse, w.b, r, threadIdx.x) = threadIdx.x ? log_sum(m[1], l[1]) : log_sum(m[0], l[0]);
}

// dλ of a head: −Σ D_2 over its rows, in a fixed order.
__global__ __launch_bounds__(1024) void diff_dlam_kernel(const float* __restrict__ d2, float* __restrict__ dlam, int64_t nb,
                                                         int accumulate, Params p) {
    __shared__ double part[16];
    const int head = blockIdx.x, j = head / p.group, g = head % p.group;
    double s = 0.0;
    for (int64_t n = threadIdx.x; n < nb * p.t; n += 1024) {
        const int64_t b = n / p.t;
        s -= d2[(b * p.hk + j) * p.rows + (n - b * p.t) * p.group + g];
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) s += __shfl_xor(s, m, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double sum = 0.0;
        for (int i = 0; i < 16; ++i) sum += part[i];
        dlam[head] = (accumulate ? dlam[head] : 0.f) + (float)sum;
    }
}

// =============================================================================
// bf16 on 32×32×16 MFMAs: dh padded to ND blocks of 32 columns, dv to 2·ND.
namespace mx {

using namespace nott::attn::mx32;
using nott::lds::barrier;
using nott::lds::dma16;
using nott::lds::dma16_at;
using nott::lds::dma4;
using nott::lds::lds_addr;
using nott::lds::wait_vm_lgkm0;

// Fills a [ROWS][32·NB] tile with the rows that `from` points to: 1 KB blocks dealt to
// WAVES waves.  WHOLE: cols is 32·NB, so no chunk is padding.
template <int NB, int ROWS, int WAVES, bool WHOLE, typename F>
__device__ __forceinline__ void fill_rows(F&& from, int cols, char NOTT_LDS* tile, int wid, int lane) {
    constexpr int CH = 4 * NB, BLOCKS = ROWS * CH / 64;
    static_assert(BLOCKS % WAVES == 0, "blocks split evenly over the waves");
#pragma unroll
    for (int qq = 0; qq < BLOCKS / WAVES; ++qq) {
        const int q = wid + WAVES * qq;
        const int i = 64 * q + lane, r = i / CH;
        const int c = swz<NB>(r, i - r * CH);   // (an involution)
        const bf16_t* src = from(r) + 8 * c;
        if constexpr (!WHOLE) {     // a select, not a branch around the address
            uint64_t a = reinterpret_cast<uint64_t>(src), z = reinterpret_cast<uint64_t>(&zero_chunk);
            asm volatile("" : "+v"(a));
            src = reinterpret_cast<const bf16_t*>(8 * c < cols ? a : z);
        }
        dma16(src, lds_addr(tile) + 1024 * q);
    }
}

// The same for tiles whose rows and columns are all there: what a lane adds to the tile's
// first row, formed once (a row's address takes some thirty cycles of vector
// multiplications, and as long again where the row's query and head are to be divided out).
template <int NB, int ROWS, int WAVES>
struct TileOffsets {
    static constexpr int CH = 4 * NB, N = ROWS * CH / 64 / WAVES;
    uint32_t v[N];
    // row(x): byte offset of the tile's row x
    template <typename F>
    __device__ __forceinline__ TileOffsets(F&& row, int wid, int lane) {
#pragma unroll
        for (int qq = 0; qq < N; ++qq) {
            const int i = 64 * (wid + WAVES * qq) + lane, x = i / CH;
            v[qq] = (uint32_t)row(x) + 16 * swz<NB>(x, i - x * CH);
        }
    }
    __device__ __forceinline__ void fill(const bf16_t* first, char NOTT_LDS* tile, int wid) const {
#pragma unroll
        for (int qq = 0; qq < N; ++qq) dma16_at(first, v[qq], lds_addr(tile) + 1024 * (wid + WAVES * qq));
    }
};

// A row as 2·NB B-operand slices: lane l holds d = 16s + 8·(l/32) + 0..7.
template <int NB, bool WHOLE>
__device__ __forceinline__ void load_row(const bf16_t* row, int cols, int lane, u32x4 (&r)[2 * NB]) {
#pragma unroll
    for (int s = 0; s < 2 * NB; ++s) {
        const int d = 16 * s + 8 * (lane >> 5);
        r[s] = *reinterpret_cast<const u32x4*>(row + (WHOLE || d < cols ? d : 0));
        if (!WHOLE && d >= cols) r[s] = u32x4{0u, 0u, 0u, 0u};
    }
}

// Where a lane reads a tile: frag_rows' and frag_cols' places, formed once.  The swizzle
// depends on a row's low 4 bits and permutes chunks within groups, so the places of other
// row blocks and groups are constants away; left to itself the compiler kept a register
// for each (61 spilled in the forward at ND = 2, 353 in the dk/dv pass at ND = 4).
template <int NB>
struct RowPlaces {
    static constexpr int K = NB % 4 == 0 ? 8 : NB % 4 == 2 ? 4 : 2;      // slices of a group
    uint32_t off[K];
    __device__ __forceinline__ explicit RowPlaces(int lane) {
#pragma unroll
        for (int s = 0; s < K; ++s) off[s] = tile_off<NB>(lane & 31, 2 * s + (lane >> 5));
    }
    __device__ __forceinline__ bf16x8 get(const char NOTT_LDS* tile, int r0, int s) const {
        return __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4 NOTT_LDS*>(tile + off[s % K] + r0 * (64 * NB) +
                                                                                   s / K * (32 * K)));
    }
};
template <int NB>
struct ColPlaces {
    static constexpr int K = NB % 4 == 0 ? 4 : NB % 4 == 2 ? 2 : 1;      // 32-column blocks of a group
    uint32_t off[K][2];
    __device__ __forceinline__ explicit ColPlaces(int lane) {
        const int j = lane & 15, g = lane >> 4, r = 4 * (g >> 1) + (j >> 2);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int col = 32 * k + 16 * (g & 1) + 4 * (j & 3);
#pragma unroll
            for (int hi = 0; hi < 2; ++hi) off[k][hi] = tile_off<NB>(r + 8 * hi, col >> 3) + (col & 7) * 2;
        }
    }
    // rows from rs (a multiple of 16), column block df
    __device__ __forceinline__ bf16x8 get(const char NOTT_LDS* tile, int rs, int df) const {
        v4i16s w[2];
#pragma unroll
        for (int hi = 0; hi < 2; ++hi)
            w[hi] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (v4i16s NOTT_LDS*)(tile + off[df % K][hi] + rs * (64 * NB) + df / K * (64 * K)));
        return __builtin_bit_cast(bf16x8, w);
    }
};

template <int NB>
__device__ __forceinline__ float dot_rows(const u32x4 (&a)[2 * NB], const u32x4 (&b)[2 * NB]) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 2 * NB; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t x = a[k][i], y = b[k][i];
            s = fmaf(__builtin_bit_cast(float, x << 16), __builtin_bit_cast(float, y << 16), s);
            s = fmaf(__builtin_bit_cast(float, x & 0xffff0000u), __builtin_bit_cast(float, y & 0xffff0000u), s);
        }
    return s + __shfl_xor(s, 32, 64);
}

// One map's step of the running softmax over TF·32 keys: the scores st become
// probabilities (packed into pb), m, l and the accumulators follow.  rel: the lane's
// visible keys, counted from its first of the tile; full: nothing is masked.
template <int TF, int NV>
__device__ __forceinline__ void softmax_step(f32x16 (&st)[TF], bf16x8 (&pb)[2 * TF], bf16x8 (&pl)[2 * TF], f32x16 (&acc)[NV], float& m, float& l,
                                             float sl2, bool full, int rel) {
    if (!full) {
#pragma unroll
        for (int f = 0; f < TF; ++f)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (!(32 * f + 8 * (r >> 2) + (r & 3) < rel)) st[f][r] = -INFINITY;
    }
    float mx = st[0][0];
#pragma unroll
    for (int f = 0; f < TF; ++f)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, st[f][r]);
    mx = max_halves(mx * sl2);   // log2 domain
    if (__any(mx > m)) {
        const float mn = fmaxf(m, mx);
        const float alpha = __builtin_amdgcn_exp2f(mn == -INFINITY ? 0.f : m - mn);
        l *= alpha;
#pragma unroll
        for (int df = 0; df < NV; ++df)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[df][e] *= alpha;
        m = mn;
    }
    const float ms = m == -INFINITY ? 0.f : m;
    float rs = 0.f;
#pragma unroll
    for (int f = 0; f < TF; ++f) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            st[f][r] = __builtin_amdgcn_exp2f(fmaf(st[f][r], sl2, -ms));
            rs += st[f][r];
        }
        pb[2 * f] = pack8(st[f], 0);
        pb[2 * f + 1] = pack8(st[f], 8);
        pl[2 * f] = pack8_lo(st[f], 0, pb[2 * f]);
        pl[2 * f + 1] = pack8_lo(st[f], 8, pb[2 * f + 1]);
    }
    l += rs;
}

template <int N>
__device__ __forceinline__ void zero(f32x16 (&a)[N]) {
#pragma unroll
    for (int f = 0; f < N; ++f)
#pragma unroll
        for (int e = 0; e < 16; ++e) a[f][e] = 0.f;
}

// 32 columns of a lane's row, as 16-byte stores: the two lanes of a row exchange 8-byte
// pieces (lane h: chunk j + h of a pair).
template <typename F>
__device__ __forceinline__ void store_block(bf16_t* row, int df, int cols, int h, F&& value) {
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
        const auto x = __builtin_amdgcn_permlane32_swap(pack_bf16x2(value(4 * j), value(4 * j + 1)),
                                                        pack_bf16x2(value(4 * j + 4), value(4 * j + 5)), false, false);
        const auto y = __builtin_amdgcn_permlane32_swap(pack_bf16x2(value(4 * j + 2), value(4 * j + 3)),
                                                        pack_bf16x2(value(4 * j + 6), value(4 * j + 7)), false, false);
        const int d = 32 * df + 8 * (j + h);
        const unsigned x0 = x[0], x1 = x[1], y0 = y[0], y1 = y[1];
        if (row && d < cols) *reinterpret_cast<u32x4*>(row + d) = u32x4{x0, y0, x1, y1};
    }
}

// Stages of ROWS keys: tiles of both maps' keys, then of the values, filled by WAVES waves.
template <int ND, int ROWS, int WAVES, bool WHOLE>
struct KeyStage {
    static constexpr int TR = ROWS, KT = TR * 64 * ND, BYTES = 4 * KT, LOADS = BYTES / 1024 / WAVES;   // loads of a wave
    const bf16_t* pk;
    const bf16_t* pv;
    TileOffsets<ND, 2 * TR, WAVES> ko;
    TileOffsets<2 * ND, TR, WAVES> vo;
    __device__ __forceinline__ KeyStage(const Params& p, const Pair& w, const bf16_t* k, const bf16_t* v, int wid, int lane)
        : pk(at(k, p.k, w.b, 0, 2 * w.j)), pv(at(v, p.v, w.b, 0, w.j)),
          ko([&](int x) { return 2 * ((x >= TR ? p.k[2] : 0) + (x >= TR ? x - TR : x) * p.k[1]); }, wid, lane),
          vo([&](int x) { return 2 * (x * p.v[1]); }, wid, lane) {}
    // keys past `most`, which nothing sees, are not read
    __device__ __forceinline__ void fill(const Params& p, int tile, int most, char NOTT_LDS* st, int wid, int lane) const {
        if (WHOLE && p.near && (tile + 1) * TR <= most) {
            ko.fill(pk + (int64_t)tile * TR * p.k[1], st, wid);
            vo.fill(pv + (int64_t)tile * TR * p.v[1], st + 2 * KT, wid);
            return;
        }
        auto key = [&](int x) { return (int64_t)min(tile * TR + x, most - 1); };
        fill_rows<ND, 2 * TR, WAVES, WHOLE>(
            [&](int x) { return pk + (x >= TR ? p.k[2] : 0) + key(x >= TR ? x - TR : x) * p.k[1]; }, p.dh, st, wid, lane);
        fill_rows<2 * ND, TR, WAVES, WHOLE>([&](int x) { return pv + key(x) * p.v[1]; }, p.dv, st + 2 * KT, wid, lane);
    }
};

// Stages of ROWS rows: tiles of both maps' queries, of dO, and the rows' statistics.
template <int ND, int ROWS, int WAVES, bool WHOLE>
struct RowStage {
    static constexpr int TR = ROWS, QT = TR * 64 * ND, BYTES = 4 * QT + 256 * 8;   // statistics: 64 floats each
    static constexpr int LOADS = 4 * QT / 1024 / WAVES;                            // beside the statistics
    const bf16_t* pq;
    const bf16_t* pd;
    const float* stats;
    bool even;              // a tile's rows are whole queries
    TileOffsets<ND, 2 * TR, WAVES> qo;
    TileOffsets<2 * ND, TR, WAVES> od;
    __device__ __forceinline__ RowStage(const Params& p, const Pair& w, const bf16_t* q, const bf16_t* dO, const float* st,
                                        int wid, int lane)
        : pq(at(q, p.q, w.b, 0, 2 * w.j * p.group)), pd(at(dO, p.od, w.b, 0, w.j * p.group)), stats(st),
          even(TR % p.group == 0),
          qo([&](int x) {
                 uint32_t i, g;
                 p.by_group.divmod(x >= TR ? x - TR : x, i, g);
                 return 2 * (i * p.q[1] + (2 * g + (x >= TR)) * p.q[2]);
             }, wid, lane),
          od([&](int x) {
                 uint32_t i, g;
                 p.by_group.divmod(x, i, g);
                 return 2 * (i * p.od[1] + g * p.od[2]);
             }, wid, lane) {}
    __device__ __forceinline__ void fill(const Params& p, const Pair& w, const bf16_t* q, const bf16_t* dO, int tile, int64_t total,
                                         char NOTT_LDS* st, int wid, int lane) const {
        const int b0 = tile * TR;
        if (WHOLE && p.near && even && b0 + TR <= p.rows) {
            const int64_t i = b0 / p.group;
            qo.fill(pq + i * p.q[1], st, wid);
            od.fill(pd + i * p.od[1], st + 2 * QT, wid);
        } else {
            auto row = [&](int x) { return RowAt(p, w, min(b0 + x, p.rows - 1)); };
            fill_rows<ND, 2 * TR, WAVES, WHOLE>(
                [&](int x) {
                    const RowAt y = row(x >= TR ? x - TR : x);
                    return at(q, p.q, w.b, y.i, 2 * y.head + (x >= TR));
                },
                p.dh, st, wid, lane);
            fill_rows<2 * ND, TR, WAVES, WHOLE>(
                [&](int x) {
                    const RowAt y = row(x);
                    return at(dO, p.od, w.b, y.i, y.head);
                },
                p.dv, st + 2 * QT, wid, lane);
        }
        const float* src = stats + min(b0 + lane, p.rows - 1);
        for (int x = wid; x < kStats; x += WAVES) dma4(src + x * total, lds_addr(st + 4 * QT) + 256 * x);
    }
};

// Forward: 128 rows a workgroup, 64 keys a stage.  A wave has 32 rows of one map (8
// waves), so that its scores and accumulator leave room for two waves a SIMD at 128 + 256
// columns and more at 64 + 128; both maps in a wave shared the values' fragments but spilled
// 41 and 213 registers (97.6 us for the benchmark's 8 x 1024 tokens, 8 heads of 64 + 128).
// The second map's output goes to the first map's waves through LDS.
template <int ND, int RING, bool WHOLE>
__global__ __launch_bounds__(128 * NW, 2) void diff_fwd32_kernel(const bf16_t* __restrict__ q, const bf16_t* __restrict__ k,
                                                                 const bf16_t* __restrict__ v, bf16_t* __restrict__ o,
                                                                 bf16_t* __restrict__ o2, float* __restrict__ lse, Params p) {
    using Keys = KeyStage<ND, 64, 2 * NW, WHOLE>;
    constexpr int NV = 2 * ND, TR = Keys::TR, KT = Keys::KT;
    extern __shared__ __attribute__((aligned(1024))) char smem_raw[];
    char NOTT_LDS* smem = (char NOTT_LDS*)smem_raw;
    const Pair w(p, blockIdx.x);
    const int nrb = (p.rows + FIXED - 1) / FIXED;
    const int r0 = (nrb - 1 - (int)blockIdx.y) * FIXED;   // heaviest (causal) blocks first
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int h = lane >> 5, map = wid / NW, wr = wid % NW;
    const int rw0 = r0 + 32 * wr, my_r = rw0 + (lane & 31);
    const RowAt r(p, w, min(my_r, p.rows - 1));
    const int vis = w.visible(p, r.i);
    const int vis_all = w.visible(p, RowAt(p, w, min(r0 + FIXED, p.rows) - 1).i);
    const int vis_lo = w.visible(p, RowAt(p, w, min(rw0, p.rows - 1)).i);
    const int vis_hi = rw0 < p.rows ? w.visible(p, RowAt(p, w, min(rw0 + 32, p.rows) - 1).i) : 0;
    const float sl2 = p.scale * kLog2e;
    const RowPlaces<ND> rows_k(lane);
    const ColPlaces<NV> cols_v(lane);
    u32x4 qr[2 * ND];
    load_row<ND, WHOLE>(at(q, p.q, w.b, r.i, 2 * r.head + map), p.dh, lane, qr);
    const Keys keys(p, w, k, v, wid, lane);
    const int nk = (vis_all + TR - 1) / TR;
#pragma unroll
    for (int i = 0; i < RING - 1; ++i)
        if (i < nk) keys.fill(p, i, vis_all, smem + i * Keys::BYTES, wid, lane);

    f32x16 acc[NV];
    zero(acc);
    float m = -INFINITY, l = 0.f;   // l: this lane's keys only
    int slot = 0, next = RING - 1;
    for (int i = 0; i < nk; ++i) {
        if (i + RING - 2 < nk) wait_vm_lgkm0<(RING - 2) * Keys::LOADS>();
        else wait_vm_lgkm0<0>();
        barrier();
        if (i + RING - 1 < nk) keys.fill(p, i + RING - 1, vis_all, smem + next * Keys::BYTES, wid, lane);
        const char NOTT_LDS* tk = smem + slot * Keys::BYTES + map * KT;
        const char NOTT_LDS* tv = smem + slot * Keys::BYTES + 2 * KT;
        slot = slot + 1 == RING ? 0 : slot + 1;
        next = next + 1 == RING ? 0 : next + 1;
        const int k0 = i * TR;
        if (k0 >= vis_hi) continue;   // every key of the block masked for this wave
        const bool full = k0 + TR <= vis_lo;
        const int rel = vis - k0 - 4 * h;
#pragma unroll
        for (int f = 0; f < 2; ++f) {
            f32x16 st[1];
            bf16x8 pb[2], pl[2];
#pragma unroll
            for (int s = 0; s < 2 * ND; ++s)
                st[0] = mfma(rows_k.get(tk, 32 * f, s), __builtin_bit_cast(bf16x8, qr[s]), s ? st[0] : f32x16{});
            softmax_step<1, NV>(st, pb, pl, acc, m, l, sl2, full, rel - 32 * f);
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int df = 0; df < NV; ++df) {
                const bf16x8 c = cols_v.get(tv, 32 * f + 16 * s, df);
                acc[df] = mfma(c, pb[s], acc[df]);
                acc[df] = mfma(c, pl[s], acc[df]);
            }
        }
    }
    l += __shfl_xor(l, 32, 64);
    const bool in = my_r < p.rows;
    const float inv = inverse(l);
    if (in && h == 0) *lse_at(p, lse, w.b, r, map) = log_sum(m, l);
    float* second = reinterpret_cast<float*>(smem_raw) + (wr * NV << 10) + lane;   // [NV][16][64] of a row block
    __syncthreads();
    if (map) {
        bf16_t* row = in && o2 ? o2 + (((int64_t)w.b * p.t + r.i) * p.h + r.head) * p.dv : nullptr;
#pragma unroll
        for (int df = 0; df < NV; ++df) {
#pragma unroll
            for (int e = 0; e < 16; ++e) second[(df * 16 + e) << 6] = acc[df][e] * inv;
            if (o2) store_block(row, df, p.dv, h, [&](int e) { return acc[df][e] * inv; });
        }
    }
    __syncthreads();
    if (map) return;
    const float lam = lambda_of(p, w.b, r);
    bf16_t* row = in ? at(o, p.o, w.b, r.i, r.head) : nullptr;
#pragma unroll
    for (int df = 0; df < NV; ++df)
        store_block(row, df, p.dv, h, [&](int e) { return acc[df][e] * inv - lam * second[(df * 16 + e) << 6]; });
}

// Few rows: 32 rows a workgroup, its keys split over the grid; 64 keys a stage, of which a
// wave takes half for one map (4 waves).
template <int ND, int RING, bool WHOLE>
__global__ __launch_bounds__(64 * NW, 1) void diff_split32_kernel(const bf16_t* __restrict__ q, const bf16_t* __restrict__ k,
                                                                  const bf16_t* __restrict__ v, Parts parts, int64_t total,
                                                                  Params p) {
    using Keys = KeyStage<ND, 64, NW, WHOLE>;
    constexpr int NV = 2 * ND, TR = Keys::TR, KT = Keys::KT;
    extern __shared__ __attribute__((aligned(1024))) char smem_raw[];
    char NOTT_LDS* smem = (char NOTT_LDS*)smem_raw;
    const Pair w(p, blockIdx.x);
    const int r0 = (int)blockIdx.z * 32;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int h = lane >> 5, map = wid >> 1, f = wid & 1;
    const int my_r = r0 + (lane & 31);
    const RowAt r(p, w, min(my_r, p.rows - 1));
    const int vis = w.visible(p, r.i);
    const int vis_lo = w.visible(p, RowAt(p, w, min(r0, p.rows - 1)).i);
    const int vis_all = w.visible(p, RowAt(p, w, min(r0 + 32, p.rows) - 1).i);
    const float sl2 = p.scale * kLog2e;
    const RowPlaces<ND> rows_k(lane);
    const ColPlaces<NV> cols_v(lane);
    u32x4 qr[2 * ND];
    load_row<ND, WHOLE>(at(q, p.q, w.b, r.i, 2 * r.head + map), p.dh, lane, qr);
    const Keys keys(p, w, k, v, wid, lane);
    const int tiles = (vis_all + TR - 1) / TR;
    const int lo = (int)((int64_t)tiles * blockIdx.y / p.nsplit), hi = (int)((int64_t)tiles * (blockIdx.y + 1) / p.nsplit);
#pragma unroll
    for (int i = 0; i < RING - 1; ++i)
        if (lo + i < hi) keys.fill(p, lo + i, vis_all, smem + i * Keys::BYTES, wid, lane);
    f32x16 acc[NV];
    zero(acc);
    float m = -INFINITY, l = 0.f;
    int slot = 0, next = RING - 1;
    for (int i = lo; i < hi; ++i) {
        if (i + RING - 2 < hi) wait_vm_lgkm0<(RING - 2) * Keys::LOADS>();
        else wait_vm_lgkm0<0>();
        barrier();
        if (i + RING - 1 < hi) keys.fill(p, i + RING - 1, vis_all, smem + next * Keys::BYTES, wid, lane);
        const char NOTT_LDS* tk = smem + slot * Keys::BYTES + map * KT;
        const char NOTT_LDS* tv = smem + slot * Keys::BYTES + 2 * KT;
        slot = slot + 1 == RING ? 0 : slot + 1;
        next = next + 1 == RING ? 0 : next + 1;
        const int k0 = i * TR + 32 * f;
        f32x16 st[1];
        bf16x8 pb[2], pl[2];
#pragma unroll
        for (int s = 0; s < 2 * ND; ++s)
            st[0] = mfma(rows_k.get(tk, 32 * f, s), __builtin_bit_cast(bf16x8, qr[s]), s ? st[0] : f32x16{});
        softmax_step<1, NV>(st, pb, pl, acc, m, l, sl2, k0 + 32 <= vis_lo, vis - k0 - 4 * h);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int df = 0; df < NV; ++df) {
                const bf16x8 c = cols_v.get(tv, 32 * f + 16 * s, df);
                acc[df] = mfma(c, pb[s], acc[df]);
                acc[df] = mfma(c, pl[s], acc[df]);
            }
    }
    // Join the halves of a map: maxima and sums, then the scaled accumulators, through LDS.
    l += __shfl_xor(l, 32, 64);
    float* sum = reinterpret_cast<float*>(smem_raw);          // [map][NV][16][64], of the second halves
    float* ml = sum + 2 * NV * 16 * 64;                       // [map][half][32][2]
    __syncthreads();
    if (h == 0) *reinterpret_cast<f32x2*>(ml + ((map * 2 + f) * 32 + (lane & 31)) * 2) = f32x2{m, l};
    __syncthreads();
    const f32x2 other = *reinterpret_cast<const f32x2*>(ml + ((map * 2 + (f ^ 1)) * 32 + (lane & 31)) * 2);
    const float top = fmaxf(m, other.x);
    const float mine = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
    const float theirs = other.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(other.x - top);
    float* half = sum + (map * NV << 10) + lane;
    if (f) {
#pragma unroll
        for (int df = 0; df < NV; ++df)
#pragma unroll
            for (int e = 0; e < 16; ++e) half[(df * 16 + e) << 6] = mine == 0.f ? 0.f : acc[df][e] * mine;
    }
    __syncthreads();
    if (f || my_r >= p.rows) return;
    const int64_t row = blockIdx.y * total + (int64_t)blockIdx.x * p.rows + my_r;
    if (h == 0) *reinterpret_cast<f32x2*>(parts.ml + (row * 2 + map) * 2) = f32x2{top, l * mine + other.y * theirs};
#pragma unroll
    for (int df = 0; df < NV; ++df)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f32x4 s4;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int x = 4 * j + e;
                s4[e] = (mine == 0.f ? 0.f : acc[df][x] * mine) + half[(df * 16 + x) << 6];
            }
            const int d = 32 * df + 8 * j + 4 * h;
            if (d < p.dv) *reinterpret_cast<f32x4*>(parts.acc + (row * 2 + map) * p.dv + d) = s4;
        }
}

// dq of both maps, and the rows' statistics: 128 rows a workgroup, 32·TF keys a stage.
template <int ND, int TF, int RING, bool WHOLE>
__global__ __launch_bounds__(64 * NW, ND <= 2 ? 2 : 1) void diff_dq32_kernel(
    const bf16_t* __restrict__ q, const bf16_t* __restrict__ k, const bf16_t* __restrict__ v, const bf16_t* __restrict__ o,
    const bf16_t* __restrict__ o2, const bf16_t* __restrict__ dO, const float* __restrict__ lse, float* __restrict__ stats,
    bf16_t* __restrict__ dq, float* __restrict__ dlam, int64_t total, Params p) {
    using Keys = KeyStage<ND, 32 * TF, NW, WHOLE>;
    constexpr int NV = 2 * ND, TR = Keys::TR, KT = Keys::KT;
    extern __shared__ __attribute__((aligned(1024))) char smem_raw[];
    char NOTT_LDS* smem = (char NOTT_LDS*)smem_raw;
    const Pair w(p, blockIdx.x);
    const int nrb = (p.rows + FIXED - 1) / FIXED;
    const int r0 = (nrb - 1 - (int)blockIdx.y) * FIXED;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int h = lane >> 5;
    const int rw0 = r0 + 32 * wid, my_r = rw0 + (lane & 31);
    const RowAt r(p, w, min(my_r, p.rows - 1));
    const int vis = w.visible(p, r.i);
    const int vis_all = w.visible(p, RowAt(p, w, min(r0 + FIXED, p.rows) - 1).i);
    const int vis_lo = w.visible(p, RowAt(p, w, min(rw0, p.rows - 1)).i);
    const int vis_hi = w.visible(p, RowAt(p, w, min(rw0 + 32, p.rows) - 1).i);
    const float sl2 = p.scale * kLog2e;
    const float lam = lambda_of(p, w.b, r);

    const RowPlaces<ND> rows_k(lane);
    const RowPlaces<NV> rows_v(lane);
    const ColPlaces<ND> cols_k(lane);
    u32x4 qr[2][2 * ND], dr[2 * NV];
#pragma unroll
    for (int m = 0; m < 2; ++m) load_row<ND, WHOLE>(at(q, p.q, w.b, r.i, 2 * r.head + m), p.dh, lane, qr[m]);
    load_row<NV, WHOLE>(at(dO, p.od, w.b, r.i, r.head), p.dv, lane, dr);
    float D[2], ls[2];
    {
        u32x4 orr[2 * NV];
        load_row<NV, WHOLE>(o2 + (((int64_t)w.b * p.t + r.i) * p.h + r.head) * p.dv, p.dv, lane, orr);
        D[1] = dot_rows<NV>(dr, orr);
        load_row<NV, WHOLE>(at(o, p.o, w.b, r.i, r.head), p.dv, lane, orr);
        D[0] = fmaf(lam, D[1], dot_rows<NV>(dr, orr));
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) ls[m] = *lse_at(p, const_cast<float*>(lse), w.b, r, m) * kLog2e;
    if (h == 0 && my_r < p.rows) {
        float* st = stats + (int64_t)blockIdx.x * p.rows + my_r;
        st[0] = ls[0];
        st[total] = ls[1];
        st[2 * total] = D[0];
        st[3 * total] = D[1];
        st[4 * total] = lam;
        if (p.token_lam) dlam[((int64_t)w.b * p.t + r.i) * p.h + r.head] = -D[1];
    }

    const int nk = (vis_all + TR - 1) / TR;
    const Keys keys(p, w, k, v, wid, lane);
#pragma unroll
    for (int i = 0; i < RING - 1; ++i)
        if (i < nk) keys.fill(p, i, vis_all, smem + i * Keys::BYTES, wid, lane);
    f32x16 adq[2][ND];
    zero(adq[0]);
    zero(adq[1]);
    int slot = 0, next = RING - 1;
    for (int i = 0; i < nk; ++i) {
        if (i + RING - 2 < nk) wait_vm_lgkm0<(RING - 2) * Keys::LOADS>();
        else wait_vm_lgkm0<0>();
        barrier();
        if (i + RING - 1 < nk) keys.fill(p, i + RING - 1, vis_all, smem + next * Keys::BYTES, wid, lane);
        const char NOTT_LDS* tk = smem + slot * Keys::BYTES;
        const char NOTT_LDS* tv = tk + 2 * KT;
        slot = slot + 1 == RING ? 0 : slot + 1;
        next = next + 1 == RING ? 0 : next + 1;
        const int k0 = i * TR;
        if (k0 >= vis_hi || rw0 >= p.rows) continue;
        const bool full = k0 + TR <= vis_lo;
        const int rel = vis - k0 - 4 * h;
#pragma unroll
        for (int f = 0; f < TF; ++f) {
            f32x16 dp;
#pragma unroll
            for (int s = 0; s < 2 * NV; ++s) dp = mfma(rows_v.get(tv, 32 * f, s), __builtin_bit_cast(bf16x8, dr[s]), s ? dp : f32x16{});
            // one map after the other (the scores of both at once spilled 10 registers at ND = 2:
            // 8 x 1024 tokens of 8 heads 107 us, 71 so)
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                f32x16 z;
#pragma unroll
                for (int s = 0; s < 2 * ND; ++s)
                    z = mfma(rows_k.get(tk + m * KT, 32 * f, s), __builtin_bit_cast(bf16x8, qr[m][s]), s ? z : f32x16{});
#pragma unroll
                for (int x = 0; x < 16; ++x) z[x] = fmaf(z[x], sl2, -ls[m]);
                if (!full) {
#pragma unroll
                    for (int x = 0; x < 16; ++x)
                        if (!(32 * f + 8 * (x >> 2) + (x & 3) < rel)) {
                            z[x] = -INFINITY;
                            dp[x] = 0.f;
                        }
                }
#pragma unroll
                for (int x = 0; x < 16; ++x)
                    z[x] = __builtin_amdgcn_exp2f(z[x]) * (m ? lam * (D[1] - dp[x]) : dp[x] - D[0]);
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const bf16x8 a = pack8(z, 8 * s), al = pack8_lo(z, 8 * s, a);
#pragma unroll
                    for (int df = 0; df < ND; ++df) {
                        const bf16x8 c = cols_k.get(tk + m * KT, 32 * f + 16 * s, df);
                        adq[m][df] = mfma(a, c, adq[m][df]);
                        adq[m][df] = mfma(al, c, adq[m][df]);
                    }
                }
            }
        }
    }
    // lane: column d = 32·df + l%32 of rows 8j + 4h + e of this wave's 32
#pragma unroll
    for (int x = 0; x < 16; ++x) {
        const int row = rw0 + 8 * (x >> 2) + 4 * h + (x & 3);
        if (row >= p.rows) continue;
        const RowAt y(p, w, row);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            bf16_t* out = at(dq, p.dq, w.b, y.i, 2 * y.head + m);
#pragma unroll
            for (int df = 0; df < ND; ++df) {
                const int d = 32 * df + (lane & 31);
                if (d < p.dh) out[d] = f32_to_bf16(adq[m][df][x] * p.scale);
            }
        }
    }
}

// dk of both maps (WHAT & 1) and dv (WHAT & 2): 128 keys a workgroup, 32·TF rows a stage,
// one share of the rows (blockIdx.z of p.nsplit; shares leave fp32 parts
// [nsplit][b·hk][s][2·dh + dv] for diff_join_keys_kernel).
template <int ND, int TF, int RING, int WHAT, bool WHOLE>
__global__ __launch_bounds__(64 * NW, WHAT == 2 && ND <= 3 ? 2 : 1) void diff_dkdv32_kernel(
    const bf16_t* __restrict__ q, const bf16_t* __restrict__ k, const bf16_t* __restrict__ v, const bf16_t* __restrict__ dO,
    const float* __restrict__ stats, bf16_t* __restrict__ dk, bf16_t* __restrict__ dv, float* __restrict__ parts, int64_t total,
    Params p) {
    constexpr bool DK = WHAT & 1, DV = WHAT & 2;
    using Rows = RowStage<ND, 32 * TF, NW, WHOLE>;
    constexpr int NV = 2 * ND, TR = Rows::TR, QT = Rows::QT;
    extern __shared__ __attribute__((aligned(1024))) char smem_raw[];
    char NOTT_LDS* smem = (char NOTT_LDS*)smem_raw;
    const Pair w(p, blockIdx.x);
    const int k0 = (int)blockIdx.y * FIXED;              // causal: the longest (first) key blocks first
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int h = lane >> 5;
    const int kw0 = k0 + 32 * wid, my_k = kw0 + (lane & 31);
    const float sl2 = p.scale * kLog2e;
    const int first = k0 < w.len ? w.first_row(p, k0) : p.rows;
    const int all = first < p.rows ? (p.rows + TR - 1) / TR - first / TR : 0;
    const int from = (int)((int64_t)all * blockIdx.z / p.nsplit), i0 = first / TR + from;
    const int nq = (int)((int64_t)all * (blockIdx.z + 1) / p.nsplit) - from;

    const RowPlaces<ND> rows_k(lane);
    const RowPlaces<NV> rows_v(lane);
    const ColPlaces<ND> cols_k(lane);
    const ColPlaces<NV> cols_v(lane);
    u32x4 kr[2][2 * ND], vr[2 * NV];
    {
        const int key = max(0, min(my_k, w.len - 1));
#pragma unroll
        for (int m = 0; m < 2; ++m) load_row<ND, WHOLE>(at(k, p.k, w.b, key, 2 * w.j + m), p.dh, lane, kr[m]);
        if (DK) load_row<NV, WHOLE>(at(v, p.v, w.b, key, w.j), p.dv, lane, vr);
    }
    const Rows rows(p, w, q, dO, stats + (int64_t)blockIdx.x * p.rows, wid, lane);
    auto issue = [&](int i, int slot) { rows.fill(p, w, q, dO, i0 + i, total, smem + slot * Rows::BYTES, wid, lane); };
#pragma unroll
    for (int i = 0; i < RING - 1; ++i)
        if (i < nq) issue(i, i);

    f32x16 adk[2][ND], adv[NV];
    zero(adk[0]);
    zero(adk[1]);
    zero(adv);
    const int lo_r = w.first_row(p, my_k), wave_lo = w.first_row(p, kw0), wave_hi = w.first_row(p, kw0 + 31);
    int slot = 0, next = RING - 1;
    for (int i = 0; i < nq; ++i) {
        // (waves with statistics to load issue more; the count of the others is a safe bound)
        if (i + RING - 2 < nq) wait_vm_lgkm0<(RING - 2) * Rows::LOADS>();
        else wait_vm_lgkm0<0>();
        barrier();
        if (i + RING - 1 < nq) issue(i + RING - 1, next);
        const char NOTT_LDS* tq = smem + slot * Rows::BYTES;
        const char NOTT_LDS* tdo = tq + 2 * QT;
        const float NOTT_LDS* ss = reinterpret_cast<const float NOTT_LDS*>(tq + 4 * QT);
        slot = slot + 1 == RING ? 0 : slot + 1;
        next = next + 1 == RING ? 0 : next + 1;
        const int b0 = (i0 + i) * TR;
        if (wave_lo >= b0 + TR || kw0 >= w.len) continue;   // no row of the block sees this wave's keys
        const bool full = b0 + TR <= p.rows && kw0 + 32 <= w.len && wave_hi <= b0;
        const int hi = my_k < w.len ? p.rows - b0 - 4 * h : -1, lo = lo_r - b0 - 4 * h;
#pragma unroll
        for (int f = 0; f < TF; ++f) {
            f32x16 t3[3];
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int s = 0; s < 2 * ND; ++s)
                    t3[m] = mfma(rows_k.get(tq + m * QT, 32 * f, s), __builtin_bit_cast(bf16x8, kr[m][s]), s ? t3[m] : f32x16{});
            if constexpr (DK)
#pragma unroll
                for (int s = 0; s < 2 * NV; ++s)
                t3[2] = mfma(rows_v.get(tdo, 32 * f, s), __builtin_bit_cast(bf16x8, vr[s]), s ? t3[2] : f32x16{});
            auto stat = [&](int which, int j) {
                return *reinterpret_cast<const f32x4 NOTT_LDS*>(ss + 64 * which + 32 * f + 8 * j + 4 * h);
            };
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f32x4 l1 = stat(0, j), l2 = stat(1, j);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    t3[0][4 * j + e] = fmaf(t3[0][4 * j + e], sl2, -l1[e]);
                    t3[1][4 * j + e] = fmaf(t3[1][4 * j + e], sl2, -l2[e]);
                }
            }
            if (!full) {
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    const int c = 32 * f + 8 * (x >> 2) + (x & 3);
                    if (!((c >= lo) & (c < hi))) {
                        t3[0][x] = t3[1][x] = -INFINITY;
                        if (DK) t3[2][x] = 0.f;
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f32x4 d1, d2;
                if (DK) d1 = stat(2, j), d2 = stat(3, j);
                const f32x4 lm = stat(4, j);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int x = 4 * j + e;
                    const float p1 = __builtin_amdgcn_exp2f(t3[0][x]), p2 = __builtin_amdgcn_exp2f(t3[1][x]) * lm[e];
                    if constexpr (DK) {
                        const float dp = t3[2][x];
                        t3[0][x] = p1 * (dp - d1[e]);
                        t3[1][x] = p2 * (d2[e] - dp);
                    }
                    if (DV) t3[2][x] = p1 - p2;
                }
            }
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                if constexpr (DK) {
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        const bf16x8 a = pack8(t3[m], 8 * s), al = pack8_lo(t3[m], 8 * s, a);
#pragma unroll
                        for (int df = 0; df < ND; ++df) {
                            const bf16x8 c = cols_k.get(tq + m * QT, 32 * f + 16 * s, df);
                            adk[m][df] = mfma(a, c, adk[m][df]);
                            adk[m][df] = mfma(al, c, adk[m][df]);
                        }
                    }
                }
                if constexpr (DV) {
                    const bf16x8 a = pack8(t3[2], 8 * s), al = pack8_lo(t3[2], 8 * s, a);
#pragma unroll
                    for (int df = 0; df < NV; ++df) {
                        const bf16x8 c = cols_v.get(tdo, 32 * f + 16 * s, df);
                        adv[df] = mfma(a, c, adv[df]);
                        adv[df] = mfma(al, c, adv[df]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int x = 0; x < 16; ++x) {
        const int key = kw0 + 8 * (x >> 2) + 4 * h + (x & 3);
        if (key >= p.s) continue;
        float* part = parts ? parts + (((int64_t)blockIdx.z * gridDim.x + blockIdx.x) * p.s + key) * (2 * p.dh + p.dv) : nullptr;
        if constexpr (DK) {
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                bf16_t* out = at(dk, p.dk, w.b, key, 2 * w.j + m);
#pragma unroll
                for (int df = 0; df < ND; ++df) {
                    const int d = 32 * df + (lane & 31);
                    if (!WHOLE && d >= p.dh) continue;
                    if (parts) part[m * p.dh + d] = adk[m][df][x] * p.scale;
                    else out[d] = f32_to_bf16(adk[m][df][x] * p.scale);
                }
            }
        }
        if constexpr (DV) {
            bf16_t* out = at(dv, p.dv_, w.b, key, w.j);
#pragma unroll
            for (int df = 0; df < NV; ++df) {
                const int d = 32 * df + (lane & 31);
                if (!WHOLE && d >= p.dv) continue;
                if (parts) part[2 * p.dh + d] = adv[df][x];
                else out[d] = f32_to_bf16(adv[df][x]);
            }
        }
    }
}

// Sums the shares of dk and dv, a thread 4 columns of a key (dh and dv are whole 8s).
__global__ __launch_bounds__(256) void diff_join_keys_kernel(const float* __restrict__ parts, bf16_t* __restrict__ dk,
                                                             bf16_t* __restrict__ dv, int64_t pairs, Params p) {
    const int per = (2 * p.dh + p.dv) / 4;
    const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (n >= pairs * p.s * per) return;
    const int64_t row = n / per;
    const int c = (int)(n - row * per) * 4;
    const f32x4 s = ordered_sum4(parts + 4 * n, pairs * p.s * per * 4, p.nsplit);
    const int bk = (int)(row / p.s), key = (int)(row - (int64_t)bk * p.s);
    const Pair w(p, bk);
    const int m = c / p.dh;
    bf16_t* out = m < 2 ? at(dk, p.dk, w.b, key, 2 * w.j + m) + (c - m * p.dh) : at(dv, p.dv_, w.b, key, w.j) + (c - 2 * p.dh);
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = f32_to_bf16(s[e]);
}

// LDS beyond the default is reserved once for each device (`done` a bit each, devices past
// 64 every time).
template <typename F>
int reserve(nott_ctx ctx, F* kernel, size_t lds, std::atomic<uint64_t>& done) {
    const uint64_t bit = ctx->device < 64 ? uint64_t(1) << ctx->device : 0;
    if (!(done.load(std::memory_order_relaxed) & bit)) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return nott::hip_fail(ctx, e, "differential attention: cannot reserve LDS");
        done.fetch_or(bit, std::memory_order_relaxed);
    }
    return NOTT_OK;
}

template <int ND, bool WHOLE>
int fwd(nott_ctx ctx, const Params& p, int64_t pairs, const bf16_t* q, const bf16_t* k, const bf16_t* v, bf16_t* o, bf16_t* o2,
        float* lse) {
    constexpr size_t lds = 2 * (size_t)KeyStage<ND, 64, 2 * NW, WHOLE>::BYTES;
    static std::atomic<uint64_t> done{0};
    auto f = &diff_fwd32_kernel<ND, 2, WHOLE>;
    if (const int st = reserve(ctx, f, lds, done); st != NOTT_OK) return st;
    hipLaunchKernelGGL(f, dim3((unsigned)pairs, (unsigned)ceil_div(p.rows, FIXED)), dim3(128 * NW), lds, ctx->stream, q, k, v,
                       o, o2, lse, p);
    return launch_status(ctx, "diff_fwd32_kernel");
}

template <int ND, bool WHOLE>
int split(nott_ctx ctx, const Params& p, int64_t pairs, const bf16_t* q, const bf16_t* k, const bf16_t* v, const Parts& parts) {
    // (two stages and two workgroups a CU: four stages and one took 69 us for 45 at 8 x 8192
    // to 16384 keys of 4 heads)
    constexpr int RING = 2;
    constexpr size_t lds = std::max<size_t>((size_t)RING * KeyStage<ND, 64, NW, WHOLE>::BYTES,
                                            (2 * 2 * ND * 16 * 64 + 2 * 2 * 32 * 2) * sizeof(float));
    static std::atomic<uint64_t> done{0};
    auto f = &diff_split32_kernel<ND, RING, WHOLE>;
    if (const int st = reserve(ctx, f, lds, done); st != NOTT_OK) return st;
    hipLaunchKernelGGL(f, dim3((unsigned)pairs, (unsigned)p.nsplit, (unsigned)ceil_div(p.rows, 32)), dim3(64 * NW), lds,
                       ctx->stream, q, k, v, parts, pairs * p.rows, p);
    return launch_status(ctx, "diff_split32_kernel");
}

template <int ND, bool WHOLE>
int bwd(nott_ctx ctx, const Params& p, int64_t pairs, const bf16_t* q, const bf16_t* k, const bf16_t* v, const bf16_t* o,
        const bf16_t* o2, const bf16_t* dO, const float* lse, float* stats, float* parts, bf16_t* dq, bf16_t* dk, bf16_t* dv,
        float* dlam) {
    // dq: 32 rows a stage (64 where a stage is 8 KB).  dk and dv: together, 64 rows a stage, as
    // long as the accumulators and operands fit a wave (64 + 128 columns: 104 us for 8 x 1024
    // tokens of 8 heads; apart 115, with 32 rows a stage 118), else apart.  A wave for each
    // map, as in the forward, forms dp twice: 125 us there, and 956 for dk alone where this
    // takes 620 (4096 tokens of 16 heads of 128 + 256).
    constexpr int TF = ND == 1 ? 2 : 1, RING = ND == 1 ? 2 : ND == 3 ? 3 : 4;
    constexpr int TFK = ND <= 2 ? 2 : 1, WHAT = ND <= 2 ? 3 : 1, TFV = ND == 3 ? 1 : 2;
    constexpr size_t lds_q = (size_t)RING * KeyStage<ND, 32 * TF, NW, WHOLE>::BYTES;
    constexpr size_t lds_kv = 2 * (size_t)RowStage<ND, 32 * TFK, NW, WHOLE>::BYTES;
    constexpr size_t lds_v = 2 * (size_t)RowStage<ND, 32 * TFV, NW, WHOLE>::BYTES;
    static std::atomic<uint64_t> done[3];
    auto fq = &diff_dq32_kernel<ND, TF, RING, WHOLE>;
    auto fk = &diff_dkdv32_kernel<ND, TFK, 2, WHAT, WHOLE>;
    if (const int st = reserve(ctx, fq, lds_q, done[0]); st != NOTT_OK) return st;
    if (const int st = reserve(ctx, fk, lds_kv, done[1]); st != NOTT_OK) return st;
    const int64_t total = pairs * p.rows;
    hipLaunchKernelGGL(fq, dim3((unsigned)pairs, (unsigned)ceil_div(p.rows, FIXED)), dim3(64 * NW), lds_q, ctx->stream, q, k, v,
                       o, o2, dO, lse, stats, dq, dlam, total, p);
    const dim3 grid((unsigned)pairs, (unsigned)ceil_div(p.s, FIXED), (unsigned)p.nsplit);
    hipLaunchKernelGGL(fk, grid, dim3(64 * NW), lds_kv, ctx->stream, q, k, v, dO, stats, dk, dv, parts, total, p);
    if constexpr (WHAT != 3) {
        auto fv = &diff_dkdv32_kernel<ND, TFV, 2, 2, WHOLE>;
        if (const int st = reserve(ctx, fv, lds_v, done[2]); st != NOTT_OK) return st;
        hipLaunchKernelGGL(fv, grid, dim3(64 * NW), lds_v, ctx->stream, q, k, v, dO, stats, dk, dv, parts, total, p);
    }
    if (parts)
        hipLaunchKernelGGL(diff_join_keys_kernel, dim3((unsigned)ceil_div(pairs * p.s * ((2 * p.dh + p.dv) / 4), 256)), dim3(256),
                           0, ctx->stream, parts, dk, dv, pairs, p);
    return launch_status(ctx, "diff_dkdv32_kernel");
}

// Blocks of 32 columns of the keys that dh and dv take (dv twice as many).
int blocks_for(const Params& p) { return (int)std::max(ceil_div(p.dh, 32), ceil_div(p.dv, 64)); }

// Calls f with that number, and whether the blocks are whole, as template arguments.
template <typename F>
int with_blocks(const Params& p, F&& f) {
    const int nd = blocks_for(p);
    auto width = [&](auto b) {
        return p.dh == 32 * nd && p.dv == 64 * nd ? f(b, std::true_type()) : f(b, std::false_type());
    };
    switch (nd) {
        case 1: return width(std::integral_constant<int, 1>());
        case 2: return width(std::integral_constant<int, 2>());
        case 3: return width(std::integral_constant<int, 3>());
        default: return width(std::integral_constant<int, 4>());
    }
}

}  // namespace mx

// =============================================================================
// 16×16 MFMAs, any element size, alignment and column count: dh padded to NS 64-byte
// slices, dv to 2·NS.  64 rows a workgroup (16 a wave), 64 keys a block; tiles are [row][d]
// in LDS, staged through registers, and second products read them by columns.
namespace any {

// 64 rows of a tile with NCH 16-byte chunks a row, loaded ahead and stored behind a barrier.
template <typename T, int NCH>
struct Stage {
    static constexpr int E = AT<T>::E, N = (BR * NCH + kThreads - 1) / kThreads;
    u32x4 r[N];
    template <typename F>
    __device__ __forceinline__ void load(F&& from, int cols, bool vec) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int t = threadIdx.x + j * kThreads;
            r[j] = t < BR * NCH ? load_chunk<T>(from(t / NCH), 0, 1, (t % NCH) * E, cols, 0, vec) : u32x4{0u, 0u, 0u, 0u};
        }
    }
    __device__ __forceinline__ void store(char* tile) const {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int t = threadIdx.x + j * kThreads;
            if (t < BR * NCH) *reinterpret_cast<u32x4*>(tile + toff(t / NCH, t % NCH, NCH)) = r[j];
        }
    }
};

// B operand of a second product: columns 16·dt.. of the rows of k-slice s (RegA's order).
template <typename T, int NCH>
__device__ __forceinline__ u32x4 columns(const char* tile, int dt, int s) {
    const int lane = threadIdx.x & 63, kq = lane >> 4;
    if constexpr (sizeof(T) == 2) {
        return frag_tr(tile, NCH, 32 * s + 4 * kq, 32 * s + 16 + 4 * kq, dt * 16);
    } else {
        const int d = dt * 16 + (lane & 15);
        f32x4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            x[e] = *reinterpret_cast<const float*>(tile + toff(16 * s + 4 * kq + e, d >> 2, NCH) + (d & 3) * 4);
        return __builtin_bit_cast(u32x4, x);
    }
}

template <typename T, int NS>
struct Dim {
    static constexpr int SL = AT<T>::SL, NV = 2 * NS;
    static constexpr int NCH = NS * 4, NCHV = NV * 4;              // chunks of a row
    static constexpr int DT = NS * SL / 16, DTV = NV * SL / 16;    // 16-column blocks
    static constexpr int KS = BR / SL;                             // k-slices of 64 rows
    static constexpr int X = BR * NCH * 16;                        // bytes of a q or k tile; v and dO take two
};

__device__ __forceinline__ void clear(f32x4& a) { a = f32x4{0.f, 0.f, 0.f, 0.f}; }

// Forward of one share of the keys (blockIdx.z of p.nsplit).
template <typename T, int NS>
__global__ __launch_bounds__(kThreads) void diff_fwd_kernel(const T* __restrict__ q, const T* __restrict__ k,
                                                            const T* __restrict__ v, T* __restrict__ o, T* __restrict__ o2,
                                                            float* __restrict__ lse, Parts parts, int64_t total, Params p) {
    using D = Dim<T, NS>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    char* lq = smem;                // both maps' q, both maps' k, v
    char* lk = smem + 2 * D::X;
    char* lv = smem + 4 * D::X;
    const Pair w(p, blockIdx.x);
    const int r0 = ((p.rows + BR - 1) / BR - 1 - (int)blockIdx.y) * BR;
    const int wid = threadIdx.x >> 6, lane = threadIdx.x & 63, r16 = lane & 15, kq = lane >> 4;
    const int my_r = r0 + wid * 16 + r16;
    const RowAt r(p, w, min(my_r, p.rows - 1));
    const int vis = w.visible(p, r.i), vis_all = w.visible(p, RowAt(p, w, min(r0 + BR, p.rows) - 1).i);
    const float sl2 = p.scale * kLog2e;
    const int tiles = (vis_all + BR - 1) / BR;
    const int lo = (int)((int64_t)tiles * blockIdx.z / p.nsplit), hi = (int)((int64_t)tiles * (blockIdx.z + 1) / p.nsplit);

    Stage<T, D::NCH> s1, s2;
    Stage<T, D::NCHV> sv;
    auto query = [&](int x, int m) {
        const RowAt y(p, w, min(r0 + x, p.rows - 1));
        return at(q, p.q, w.b, y.i, 2 * y.head + m);
    };
    s1.load([&](int x) { return query(x, 0); }, p.dh, p.vec);
    s2.load([&](int x) { return query(x, 1); }, p.dh, p.vec);
    s1.store(lq);
    s2.store(lq + D::X);
    auto load = [&](int tile) {
        auto key = [&](int x) { return min(tile * BR + x, vis_all - 1); };
        s1.load([&](int x) { return at(k, p.k, w.b, key(x), 2 * w.j); }, p.dh, p.vec);
        s2.load([&](int x) { return at(k, p.k, w.b, key(x), 2 * w.j + 1); }, p.dh, p.vec);
        sv.load([&](int x) { return at(v, p.v, w.b, key(x), w.j); }, p.dv, p.vec);
    };
    f32x4 acc[2][D::DTV];
#pragma unroll
    for (int i = 0; i < D::DTV; ++i) {
        clear(acc[0][i]);
        clear(acc[1][i]);
    }
    float mm[2] = {-INFINITY, -INFINITY}, ll[2] = {0.f, 0.f};
    if (lo < hi) load(lo);
    for (int tile = lo; tile < hi; ++tile) {
        __syncthreads();
        s1.store(lk);
        s2.store(lk + D::X);
        sv.store(lv);
        __syncthreads();
        if (tile + 1 < hi) load(tile + 1);
        const int k0 = tile * BR;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            f32x4 sc[4];    // lane: its row's scores of keys k0 + 16·kt + 4·kq + e
            float mx = -INFINITY;
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                clear(sc[kt]);
#pragma unroll
                for (int s = 0; s < NS; ++s)
                    mma<T>(frag(lk + m * D::X, kt * 16, s, D::NCH), frag(lq + m * D::X, wid * 16, s, D::NCH), sc[kt]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sc[kt][e] = k0 + kt * 16 + kq * 4 + e < vis ? sc[kt][e] * sl2 : -INFINITY;
                    mx = fmaxf(mx, sc[kt][e]);
                }
            }
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const float mn = fmaxf(mm[m], mx), ms = mn == -INFINITY ? 0.f : mn;
            const float alpha = __builtin_amdgcn_exp2f(mm[m] - ms);
            float rs = 0.f;
#pragma unroll
            for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sc[kt][e] = __builtin_amdgcn_exp2f(sc[kt][e] - ms);
                    rs += sc[kt][e];
                }
            rs += __shfl_xor(rs, 16, 64);
            rs += __shfl_xor(rs, 32, 64);
            ll[m] = ll[m] * alpha + rs;
            mm[m] = mn;
            float al[4];    // accumulator rows are 4·kq + e
#pragma unroll
            for (int e = 0; e < 4; ++e) al[e] = __shfl(alpha, kq * 4 + e, 64);
#pragma unroll
            for (int dt = 0; dt < D::DTV; ++dt)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[m][dt][e] *= al[e];
            const RegA<T, true> pa(sc);
#pragma unroll
            for (int s = 0; s < D::KS; ++s)
#pragma unroll
                for (int dt = 0; dt < D::DTV; ++dt) pa.mma(s, columns<T, D::NCHV>(lv, dt, s), acc[m][dt]);
        }
    }
    if (parts.acc) {
        const int64_t base = blockIdx.z * total + (int64_t)blockIdx.x * p.rows;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int row = r0 + wid * 16 + kq * 4 + e;
            if (row >= p.rows) continue;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int dt = 0; dt < D::DTV; ++dt) {
                    const int d = dt * 16 + r16;
                    if (d < p.dv) parts.acc[((base + row) * 2 + m) * p.dv + d] = acc[m][dt][e];
                }
        }
        if (kq < 2 && my_r < p.rows) {
            float* out = parts.ml + ((base + my_r) * 2 + kq) * 2;
            out[0] = kq ? mm[1] : mm[0];
            out[1] = kq ? ll[1] : ll[0];
        }
        return;
    }
    const float i1 = inverse(ll[0]), i2 = inverse(ll[1]);
    const float lam = lambda_of(p, w.b, r);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float a1 = __shfl(i1, kq * 4 + e, 64), a2 = __shfl(i2, kq * 4 + e, 64), lm = __shfl(lam, kq * 4 + e, 64);
        const int row = r0 + wid * 16 + kq * 4 + e;
        if (row >= p.rows) continue;
        const RowAt y(p, w, row);
        T* po = at(o, p.o, w.b, y.i, y.head);
        const int64_t second = (((int64_t)w.b * p.t + y.i) * p.h + y.head) * p.dv;
#pragma unroll
        for (int dt = 0; dt < D::DTV; ++dt) {
            const int d = dt * 16 + r16;
            if (d >= p.dv) continue;
            const float b = acc[1][dt][e] * a2;
            Io<T>::st(po, d, acc[0][dt][e] * a1 - lm * b);
            if (o2) Io<T>::st(o2, second + d, b);
        }
    }
    if (kq < 2 && my_r < p.rows) *lse_at(p, lse, w.b, r, kq) = log_sum(kq ? mm[1] : mm[0], kq ? ll[1] : ll[0]);
}

// Rows' statistics (kStats above), a wave a row.
template <typename T>
__global__ __launch_bounds__(256) void diff_stats_kernel(const T* __restrict__ o, const T* __restrict__ o2,
                                                         const T* __restrict__ dO, const float* __restrict__ lse,
                                                         float* __restrict__ stats, float* __restrict__ dlam, int64_t total,
                                                         Params p) {
    const int lane = threadIdx.x & 63;
    for (int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); n < total; n += (int64_t)gridDim.x * 4) {
        const int bk = (int)(n / p.rows);
        const Pair w(p, bk);
        const RowAt r(p, w, (int)(n - (int64_t)bk * p.rows));
        const int64_t second = (((int64_t)w.b * p.t + r.i) * p.h + r.head) * p.dv;
        const T* po = at(o, p.o, w.b, r.i, r.head);
        const T* pd = at(dO, p.od, w.b, r.i, r.head);
        float a = 0.f, b = 0.f;
        for (int d = lane; d < p.dv; d += 64) {
            const float g = Io<T>::ld(pd, d);
            a = fmaf(g, Io<T>::ld(po, d), a);
            b = fmaf(g, Io<T>::ld(o2, second + d), b);
        }
        a = wave_sum(a);
        b = wave_sum(b);
        if (lane) continue;
        const float lam = lambda_of(p, w.b, r);
        stats[n] = *lse_at(p, const_cast<float*>(lse), w.b, r, 0) * kLog2e;
        stats[total + n] = *lse_at(p, const_cast<float*>(lse), w.b, r, 1) * kLog2e;
        stats[2 * total + n] = fmaf(lam, b, a);
        stats[3 * total + n] = b;
        stats[4 * total + n] = lam;
        if (p.token_lam) dlam[((int64_t)w.b * p.t + r.i) * p.h + r.head] = -b;
    }
}

template <typename T, int NS>
__global__ __launch_bounds__(kThreads) void diff_dq_kernel(const T* __restrict__ q, const T* __restrict__ k,
                                                           const T* __restrict__ v, const T* __restrict__ dO,
                                                           const float* __restrict__ stats, T* __restrict__ dq, int64_t total,
                                                           Params p) {
    using D = Dim<T, NS>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    char* lq = smem;                // q of both maps, dO, k of both maps, v
    char* ldo = smem + 2 * D::X;
    char* lk = smem + 4 * D::X;
    char* lv = smem + 6 * D::X;
    const Pair w(p, blockIdx.x);
    const int r0 = ((p.rows + BR - 1) / BR - 1 - (int)blockIdx.y) * BR;
    const int wid = threadIdx.x >> 6, lane = threadIdx.x & 63, r16 = lane & 15, kq = lane >> 4;
    const int my_r = min(r0 + wid * 16 + r16, p.rows - 1);
    const int vis = w.visible(p, RowAt(p, w, my_r).i), vis_all = w.visible(p, RowAt(p, w, min(r0 + BR, p.rows) - 1).i);
    const float sl2 = p.scale * kLog2e;
    float st[kStats];
#pragma unroll
    for (int x = 0; x < kStats; ++x) st[x] = stats[x * total + (int64_t)blockIdx.x * p.rows + my_r];
    Stage<T, D::NCH> s1, s2;
    Stage<T, D::NCHV> sv;
    auto row = [&](int x) { return RowAt(p, w, min(r0 + x, p.rows - 1)); };
    s1.load([&](int x) { const RowAt y = row(x); return at(q, p.q, w.b, y.i, 2 * y.head); }, p.dh, p.vec);
    s2.load([&](int x) { const RowAt y = row(x); return at(q, p.q, w.b, y.i, 2 * y.head + 1); }, p.dh, p.vec);
    sv.load([&](int x) { const RowAt y = row(x); return at(dO, p.od, w.b, y.i, y.head); }, p.dv, p.vec);
    s1.store(lq);
    s2.store(lq + D::X);
    sv.store(ldo);
    auto load = [&](int tile) {
        auto key = [&](int x) { return min(tile * BR + x, vis_all - 1); };
        s1.load([&](int x) { return at(k, p.k, w.b, key(x), 2 * w.j); }, p.dh, p.vec);
        s2.load([&](int x) { return at(k, p.k, w.b, key(x), 2 * w.j + 1); }, p.dh, p.vec);
        sv.load([&](int x) { return at(v, p.v, w.b, key(x), w.j); }, p.dv, p.vec);
    };
    f32x4 acc[2][D::DT];
#pragma unroll
    for (int i = 0; i < D::DT; ++i) {
        clear(acc[0][i]);
        clear(acc[1][i]);
    }
    const int tiles = (vis_all + BR - 1) / BR;
    if (tiles) load(0);
    for (int tile = 0; tile < tiles; ++tile) {
        __syncthreads();
        s1.store(lk);
        s2.store(lk + D::X);
        sv.store(lv);
        __syncthreads();
        if (tile + 1 < tiles) load(tile + 1);
        f32x4 z[2][4];
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
            f32x4 dp;
            clear(dp);
#pragma unroll
            for (int s = 0; s < D::NV; ++s) mma<T>(frag(lv, kt * 16, s, D::NCHV), frag(ldo, wid * 16, s, D::NCHV), dp);
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                clear(z[m][kt]);
#pragma unroll
                for (int s = 0; s < NS; ++s)
                    mma<T>(frag(lk + m * D::X, kt * 16, s, D::NCH), frag(lq + m * D::X, wid * 16, s, D::NCH), z[m][kt]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool ok = tile * BR + kt * 16 + kq * 4 + e < vis;
                    const float pe = __builtin_amdgcn_exp2f(ok ? fmaf(z[m][kt][e], sl2, -st[m]) : -INFINITY);
                    const float x = ok ? dp[e] : 0.f;
                    z[m][kt][e] = pe * (m ? st[4] * (st[3] - x) : x - st[2]);
                }
            }
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const RegA<T, true> a(z[m]);
#pragma unroll
            for (int s = 0; s < D::KS; ++s)
#pragma unroll
                for (int dt = 0; dt < D::DT; ++dt) a.mma(s, columns<T, D::NCH>(lk + m * D::X, dt, s), acc[m][dt]);
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int x = r0 + wid * 16 + kq * 4 + e;
        if (x >= p.rows) continue;
        const RowAt y(p, w, x);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            T* out = at(dq, p.dq, w.b, y.i, 2 * y.head + m);
#pragma unroll
            for (int dt = 0; dt < D::DT; ++dt)
                if (dt * 16 + r16 < p.dh) Io<T>::st(out, dt * 16 + r16, acc[m][dt][e] * p.scale);
        }
    }
}

template <typename T, int NS>
__global__ __launch_bounds__(kThreads) void diff_dkdv_kernel(const T* __restrict__ q, const T* __restrict__ k,
                                                             const T* __restrict__ v, const T* __restrict__ dO,
                                                             const float* __restrict__ stats, T* __restrict__ dk,
                                                             T* __restrict__ dv, int64_t total, Params p) {
    using D = Dim<T, NS>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    char* lk = smem;                // k of both maps, v, q of both maps, dO, statistics
    char* lv = smem + 2 * D::X;
    char* lq = smem + 4 * D::X;
    char* ldo = smem + 6 * D::X;
    float* ls = reinterpret_cast<float*>(smem + 8 * D::X);
    const Pair w(p, blockIdx.x);
    const int k0 = (int)blockIdx.y * BR;
    const int wid = threadIdx.x >> 6, lane = threadIdx.x & 63, r16 = lane & 15, kq = lane >> 4;
    const int my_k = k0 + wid * 16 + r16;
    const float sl2 = p.scale * kLog2e;
    Stage<T, D::NCH> s1, s2;
    Stage<T, D::NCHV> sv;
    auto key = [&](int x) { return max(0, min(k0 + x, w.len - 1)); };
    s1.load([&](int x) { return at(k, p.k, w.b, key(x), 2 * w.j); }, p.dh, p.vec);
    s2.load([&](int x) { return at(k, p.k, w.b, key(x), 2 * w.j + 1); }, p.dh, p.vec);
    sv.load([&](int x) { return at(v, p.v, w.b, key(x), w.j); }, p.dv, p.vec);
    s1.store(lk);
    s2.store(lk + D::X);
    sv.store(lv);
    const int first = k0 < w.len ? w.first_row(p, k0) : p.rows;
    const int lo_r = w.first_row(p, my_k);
    const int t0 = first / BR, t1 = first < p.rows ? (p.rows + BR - 1) / BR : t0;
    float nst[2] = {0.f, 0.f};
    auto load = [&](int tile) {
        auto row = [&](int x) { return RowAt(p, w, min(tile * BR + x, p.rows - 1)); };
        s1.load([&](int x) { const RowAt y = row(x); return at(q, p.q, w.b, y.i, 2 * y.head); }, p.dh, p.vec);
        s2.load([&](int x) { const RowAt y = row(x); return at(q, p.q, w.b, y.i, 2 * y.head + 1); }, p.dh, p.vec);
        sv.load([&](int x) { const RowAt y = row(x); return at(dO, p.od, w.b, y.i, y.head); }, p.dv, p.vec);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int n = threadIdx.x + x * kThreads;
            if (n < kStats * BR)
                nst[x] = stats[(n / BR) * total + (int64_t)blockIdx.x * p.rows + min(tile * BR + n % BR, p.rows - 1)];
        }
    };
    f32x4 adk[2][D::DT], adv[D::DTV];
#pragma unroll
    for (int i = 0; i < D::DT; ++i) {
        clear(adk[0][i]);
        clear(adk[1][i]);
    }
#pragma unroll
    for (int i = 0; i < D::DTV; ++i) clear(adv[i]);
    if (t0 < t1) load(t0);
    for (int tile = t0; tile < t1; ++tile) {
        __syncthreads();
        s1.store(lq);
        s2.store(lq + D::X);
        sv.store(ldo);
#pragma unroll
        for (int x = 0; x < 2; ++x)
            if (threadIdx.x + x * kThreads < kStats * BR) ls[threadIdx.x + x * kThreads] = nst[x];
        __syncthreads();
        if (tile + 1 < t1) load(tile + 1);
        f32x4 z[2][4], pw[4];
#pragma unroll
        for (int qt = 0; qt < 4; ++qt) {
            f32x4 dp;
            clear(dp);
            clear(pw[qt]);
#pragma unroll
            for (int s = 0; s < D::NV; ++s) mma<T>(frag(ldo, qt * 16, s, D::NCHV), frag(lv, wid * 16, s, D::NCHV), dp);
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                clear(z[m][qt]);
#pragma unroll
                for (int s = 0; s < NS; ++s)
                    mma<T>(frag(lq + m * D::X, qt * 16, s, D::NCH), frag(lk + m * D::X, wid * 16, s, D::NCH), z[m][qt]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int rl = qt * 16 + kq * 4 + e, row = tile * BR + rl;
                    const bool ok = (row < p.rows) & (my_k < w.len) & (row >= lo_r);
                    const float pe = __builtin_amdgcn_exp2f(ok ? fmaf(z[m][qt][e], sl2, -ls[m * BR + rl]) : -INFINITY);
                    const float x = ok ? dp[e] : 0.f, lam = ls[4 * BR + rl];
                    z[m][qt][e] = pe * (m ? lam * (ls[3 * BR + rl] - x) : x - ls[2 * BR + rl]);
                    pw[qt][e] += m ? -lam * pe : pe;
                }
            }
        }
        const RegA<T, true> a0(z[0]), a1(z[1]), aw(pw);
#pragma unroll
        for (int s = 0; s < D::KS; ++s) {
#pragma unroll
            for (int dt = 0; dt < D::DT; ++dt) {
                a0.mma(s, columns<T, D::NCH>(lq, dt, s), adk[0][dt]);
                a1.mma(s, columns<T, D::NCH>(lq + D::X, dt, s), adk[1][dt]);
            }
#pragma unroll
            for (int dt = 0; dt < D::DTV; ++dt) aw.mma(s, columns<T, D::NCHV>(ldo, dt, s), adv[dt]);
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int x = k0 + wid * 16 + kq * 4 + e;
        if (x >= p.s) continue;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            T* out = at(dk, p.dk, w.b, x, 2 * w.j + m);
#pragma unroll
            for (int dt = 0; dt < D::DT; ++dt)
                if (dt * 16 + r16 < p.dh) Io<T>::st(out, dt * 16 + r16, adk[m][dt][e] * p.scale);
        }
        T* out = at(dv, p.dv_, w.b, x, w.j);
#pragma unroll
        for (int dt = 0; dt < D::DTV; ++dt)
            if (dt * 16 + r16 < p.dv) Io<T>::st(out, dt * 16 + r16, adv[dt][e]);
    }
}

template <typename T, int NS>
int fwd(nott_ctx ctx, const Params& p, int64_t pairs, const T* q, const T* k, const T* v, T* o, T* o2, float* lse,
        const Parts& parts) {
    constexpr size_t lds = 6 * Dim<T, NS>::X;
    static std::atomic<uint64_t> done{0};
    auto f = &diff_fwd_kernel<T, NS>;
    if (const int st = mx::reserve(ctx, f, lds, done); st != NOTT_OK) return st;
    hipLaunchKernelGGL(f, dim3((unsigned)pairs, (unsigned)ceil_div(p.rows, BR), (unsigned)p.nsplit), dim3(kThreads), lds,
                       ctx->stream, q, k, v, o, o2, lse, parts, pairs * p.rows, p);
    return launch_status(ctx, "diff_fwd_kernel");
}

template <typename T, int NS>
int bwd(nott_ctx ctx, const Params& p, int64_t pairs, const T* q, const T* k, const T* v, const T* o, const T* o2, const T* dO,
        const float* lse, float* stats, T* dq, T* dk, T* dv, float* dlam) {
    constexpr size_t lds_q = 8 * Dim<T, NS>::X, lds_kv = lds_q + kStats * BR * sizeof(float);
    static std::atomic<uint64_t> done[2];
    auto fq = &diff_dq_kernel<T, NS>;
    auto fk = &diff_dkdv_kernel<T, NS>;
    if (const int st = mx::reserve(ctx, fq, lds_q, done[0]); st != NOTT_OK) return st;
    if (const int st = mx::reserve(ctx, fk, lds_kv, done[1]); st != NOTT_OK) return st;
    const int64_t total = pairs * p.rows;
    hipLaunchKernelGGL(diff_stats_kernel<T>, dim3((unsigned)std::min<int64_t>(ceil_div(total, 4), kMostBlocks)), dim3(256), 0,
                       ctx->stream, o, o2, dO, lse, stats, dlam, total, p);
    hipLaunchKernelGGL(fq, dim3((unsigned)pairs, (unsigned)ceil_div(p.rows, BR)), dim3(kThreads), lds_q, ctx->stream, q, k, v,
                       dO, stats, dq, total, p);
    hipLaunchKernelGGL(fk, dim3((unsigned)pairs, (unsigned)ceil_div(p.s, BR)), dim3(kThreads), lds_kv, ctx->stream, q, k, v, dO,
                       stats, dk, dv, total, p);
    return launch_status(ctx, "diff_dkdv_kernel");
}

}  // namespace any

bool even16(const void* p, const int64_t (&st)[3], int elem) {
    return (uintptr_t)p % 16 == 0 && st[0] * elem % 16 == 0 && st[1] * elem % 16 == 0 && st[2] * elem % 16 == 0;
}

int check(nott_ctx ctx, const nott_diff_attn_desc* d, nott_dtype dtype, Params* p) {
    NOTT_REQUIRE(ctx, nott::valid_dtype(dtype), "differential attention: bad dtype");
    NOTT_REQUIRE(ctx, d != nullptr, "differential attention: null descriptor");
    NOTT_REQUIRE(ctx, d->b >= 0 && d->h >= 0 && d->hk >= 0 && d->t >= 0 && d->s >= 0 && d->dh > 0 && d->dv > 0,
                 "differential attention: bad shape");
    NOTT_REQUIRE(ctx, d->h == 0 || (d->hk > 0 && d->h % d->hk == 0), "differential attention: heads must be a multiple of key heads");
    const int most = dtype == NOTT_BF16 ? 128 : 64;
    NOTT_REQUIRE(ctx, d->dh <= most && d->dv <= 2 * most,
                 "differential attention: head dim above 128 (bf16) / 64 (fp32), or values' above twice that, is not supported");
    NOTT_REQUIRE(ctx, d->scale > 0.0 && d->scale < 1e30, "differential attention: scale must be positive");
    NOTT_REQUIRE(ctx, (d->causal | d->token_lam) >> 1 == 0, "differential attention: causal and token_lam are 0 or 1");
    const int64_t group = d->h ? d->h / d->hk : 1;      // (without heads nothing is computed, but FastDiv divides by it)
    NOTT_REQUIRE(ctx, d->b * std::max<int64_t>(d->hk, 1) < (int64_t(1) << 23) && d->h < (int64_t(1) << 20) &&
                          d->t * group <= 4000000 && d->s <= 4000000,
                 "differential attention: too many heads or too long a sequence");
    p->t = (int32_t)d->t; p->s = (int32_t)d->s; p->dh = (int32_t)d->dh; p->dv = (int32_t)d->dv;
    p->h = (int32_t)d->h; p->hk = (int32_t)d->hk; p->group = (int32_t)group; p->rows = (int32_t)(d->t * group);
    p->causal = d->causal; p->token_lam = d->token_lam;
    p->scale = (float)d->scale;
    p->by_group = FastDiv((uint32_t)group);
    p->nsplit = 1;
    auto strides = [&](const int64_t (&in)[3], int64_t (&out)[3], int64_t rows, int64_t heads, int64_t width) {
        const bool dense = in[0] == 0 && in[1] == 0 && in[2] == 0;
        out[0] = dense ? rows * heads * width : in[0];
        out[1] = dense ? heads * width : in[1];
        out[2] = dense ? width : in[2];
    };
    strides(d->q_stride, p->q, d->t, 2 * d->h, d->dh);
    strides(d->k_stride, p->k, d->s, 2 * d->hk, d->dh);
    strides(d->v_stride, p->v, d->s, d->hk, d->dv);
    strides(d->o_stride, p->o, d->t, d->h, d->dv);
    strides(d->do_stride, p->od, d->t, d->h, d->dv);
    strides(d->dq_stride, p->dq, d->t, 2 * d->h, d->dh);
    strides(d->dk_stride, p->dk, d->s, 2 * d->hk, d->dh);
    strides(d->dv_stride, p->dv_, d->s, d->hk, d->dv);
    p->near = 1;
    for (const auto* x : {&p->q, &p->k, &p->v, &p->od})
        p->near &= (*x)[1] >= 0 && (*x)[2] >= 0 && (*x)[1] < (int64_t(1) << 21) && (*x)[2] * 2 * (group + 1) < (int64_t(1) << 28);
    return NOTT_OK;
}

// 64-byte slices, a power of two.
int slices_for(const Params& p, int sl) {
    const int need = (int)std::max(ceil_div(p.dh, sl), ceil_div(p.dv, 2 * sl));
    return need <= 1 ? 1 : need <= 2 ? 2 : 4;
}

// Rows that nothing was computed for: zeros over a strided [b, rows, heads, width] tensor.
__global__ __launch_bounds__(256) void diff_zero_kernel(uint16_t* __restrict__ p16, float* __restrict__ p32, int64_t n,
                                                        int64_t rows, int64_t heads, int64_t width, int64_t sb, int64_t st,
                                                        int64_t sh, float value) {
    for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < n; x += (int64_t)gridDim.x * 256) {
        int64_t i = x;
        const int64_t d = i % width;
        i /= width;
        const int64_t hd = i % heads;
        i /= heads;
        const int64_t at = i / rows * sb + i % rows * st + hd * sh + d;
        if (p16) p16[at] = 0;
        else p32[at] = value;
    }
}
int fill(nott_ctx ctx, nott_dtype dtype, void* dst, int64_t b, int64_t rows, int64_t heads, int64_t width,
         const int64_t (&st)[3], float value = 0.f) {
    const int64_t n = b * rows * heads * width;
    if (n == 0) return NOTT_OK;
    NOTT_REQUIRE(ctx, dst != nullptr, "differential attention: null buffer");
    hipLaunchKernelGGL(diff_zero_kernel, dim3((unsigned)std::min<int64_t>(ceil_div(n, 256), kMostBlocks)), dim3(256), 0, ctx->stream,
                       dtype == NOTT_BF16 ? static_cast<uint16_t*>(dst) : nullptr,
                       dtype == NOTT_BF16 ? nullptr : static_cast<float*>(dst), n, rows, heads, width, st[0], st[1], st[2], value);
    return launch_status(ctx, "diff_zero_kernel");
}

template <typename T>
int join(nott_ctx ctx, const Params& p, int64_t pairs, const Parts& parts, T* o, T* o2, float* lse) {
    const int64_t total = pairs * p.rows;
    if (p.nsplit <= 4)
        hipLaunchKernelGGL((diff_join_kernel<T, 1>), dim3((unsigned)total), dim3(64), 0, ctx->stream, parts, o, o2, lse, total, p);
    else
        hipLaunchKernelGGL((diff_join_kernel<T, 4>), dim3((unsigned)total), dim3(256), 0, ctx->stream, parts, o, o2, lse, total, p);
    return launch_status(ctx, "diff_join_kernel");
}

// Room for nsplit parts, or none.
Parts parts_for(nott_ctx ctx, const Params& p, int64_t pairs, int64_t nsplit) {
    const int64_t rows = nsplit * pairs * p.rows * 2, acc = (rows * p.dv + 3) & ~int64_t(3);   // {m, l} are read by 16 bytes
    float* w = static_cast<float*>(nott::optional_workspace(ctx, (size_t)(acc + rows * 2) * sizeof(float)));
    return {w, w ? w + acc : nullptr};
}

}  // namespace

extern "C" int nott_diff_attention_fwd(nott_ctx ctx, const nott_diff_attn_desc* d, nott_dtype dtype, const void* q,
                                       const void* k, const void* v, const float* lam, const int32_t* lengths,
                                       const int32_t* q_start, void* o, float* lse, void* o2) {
    NOTT_CHECK_CTX(ctx);
    Params p{};
    if (const int st = check(ctx, d, dtype, &p); st != NOTT_OK) return st;
    if (d->b * d->h * d->t == 0) return NOTT_OK;
    nott::DeviceScope scope(ctx->device);
    NOTT_REQUIRE(ctx, q && o && lse && lam, "nott_diff_attention_fwd: null buffer");
    if (d->s == 0) {    // no keys: nothing to attend to
        if (const int st = fill(ctx, dtype, o, d->b, d->t, d->h, d->dv, p.o); st != NOTT_OK) return st;
        const int64_t dense2[3] = {d->t * d->h * d->dv, d->h * d->dv, d->dv}, one[3] = {2 * d->h * d->t, 1, d->t};
        if (o2)
            if (const int st = fill(ctx, dtype, o2, d->b, d->t, d->h, d->dv, dense2); st != NOTT_OK) return st;
        return fill(ctx, NOTT_F32, lse, d->b, d->t, 2 * d->h, 1, one, -INFINITY);
    }
    NOTT_REQUIRE(ctx, k && v, "nott_diff_attention_fwd: null buffer");
    p.lam = lam;
    p.lengths = lengths;
    p.start = q_start;
    const int elem = (int)nott::dtype_size(dtype);
    p.vec = even16(q, p.q, elem) && even16(k, p.k, elem) && even16(v, p.v, elem);
    const int64_t pairs = d->b * d->hk;
    if (dtype == NOTT_BF16 && p.vec && p.dh % 8 == 0 && p.dv % 8 == 0 && even16(o, p.o, 2) && (uintptr_t)o2 % 16 == 0) {
        const auto* tq = static_cast<const bf16_t*>(q);
        const auto* tk = static_cast<const bf16_t*>(k);
        const auto* tv = static_cast<const bf16_t*>(v);
        auto* to = static_cast<bf16_t*>(o);
        auto* to2 = static_cast<bf16_t*>(o2);
        // Fewer workgroups than half the CUs: keys split, if there are two parts or more (128
        // rows against 8192 keys, 8 heads: 212 us whole, 30 split; 1024 tokens of 16 heads on 4 in
        // one part 52 us, whole 38).
        if (2 * pairs * ceil_div(p.rows, mx::FIXED) <= ctx->num_cu && p.s >= 256 && ceil_div(p.rows, 32) <= 65535) {
            const int64_t per = 64 * 4;     // keys to a workgroup at the least
            const int64_t most = std::min<int64_t>(kMostParts, ceil_div(p.s, per));
            const int64_t n = std::min<int64_t>(most, ceil_div(2 * ctx->num_cu, pairs * ceil_div(p.rows, 32)));
            const Parts parts = n > 1 ? parts_for(ctx, p, pairs, n) : Parts{};
            if (parts.acc) {
                p.nsplit = (int32_t)n;
                const int st = mx::with_blocks(p, [&](auto b, auto w) {
                    return mx::split<decltype(b)::value, decltype(w)::value>(ctx, p, pairs, tq, tk, tv, parts);
                });
                return st != NOTT_OK ? st : join(ctx, p, pairs, parts, to, to2, lse);
            }
        }
        return mx::with_blocks(p, [&](auto b, auto w) {
            return mx::fwd<decltype(b)::value, decltype(w)::value>(ctx, p, pairs, tq, tk, tv, to, to2, lse);
        });
    }
    auto run = [&](auto type) {
        using T = decltype(type);
        const auto* tq = static_cast<const T*>(q);
        const auto* tk = static_cast<const T*>(k);
        const auto* tv = static_cast<const T*>(v);
        auto* to = static_cast<T*>(o);
        auto* to2 = static_cast<T*>(o2);
        Parts parts{};
        const int64_t groups = pairs * ceil_div(p.rows, BR);
        // Fewer workgroups than CUs, or where all keys are seen than three of four: keys split.
        // Split against whole, fp32 and unaligned bf16, 16 + 32 to 64 + 128 columns: causal (blocks
        // differ in length, and parts even that out) 0.5 to 0.8 of the time at 72 to 168
        // workgroups, 0.8 to 0.95 at 195 to 240 (at 16 + 32 columns in fp32 up to 1.1); all keys
        // seen 0.5 to 0.8 up to 128, 0.8 to 1.1 at 144 to 168, 1.05 to 1.3 from 195 on, where
        // the parts run in a second round.
        if (groups < (p.causal ? ctx->num_cu : ctx->num_cu * 3 / 4) && p.s >= 512) {
            const int64_t most = std::min<int64_t>(kMostParts, ceil_div(p.s, 4 * BR));
            const int64_t n = std::min<int64_t>(most, ceil_div(2 * ctx->num_cu, groups));
            if (n > 1) parts = parts_for(ctx, p, pairs, n);
            if (parts.acc) p.nsplit = (int32_t)n;
        }
        const int ns = slices_for(p, AT<T>::SL);
        const int st = ns == 1   ? any::fwd<T, 1>(ctx, p, pairs, tq, tk, tv, to, to2, lse, parts)
                       : ns == 2 ? any::fwd<T, 2>(ctx, p, pairs, tq, tk, tv, to, to2, lse, parts)
                                 : any::fwd<T, 4>(ctx, p, pairs, tq, tk, tv, to, to2, lse, parts);
        return st != NOTT_OK || !parts.acc ? st : join(ctx, p, pairs, parts, to, to2, lse);
    };
    return dtype == NOTT_BF16 ? run(bf16_t()) : run(float());
}

extern "C" int nott_diff_attention_bwd(nott_ctx ctx, const nott_diff_attn_desc* d, nott_dtype dtype, const void* dO,
                                       const void* q, const void* k, const void* v, const float* lam, const int32_t* lengths,
                                       const int32_t* q_start, const void* o, const void* o2, const float* lse, void* dq,
                                       void* dk, void* dv, float* dlam, int accumulate) {
    NOTT_CHECK_CTX(ctx);
    Params p{};
    if (const int st = check(ctx, d, dtype, &p); st != NOTT_OK) return st;
    nott::DeviceScope scope(ctx->device);
    NOTT_REQUIRE(ctx, !(accumulate && d->token_lam), "nott_diff_attention_bwd: accumulate goes with one lambda a head");
    if (d->b == 0 || d->h == 0 || d->t == 0 || d->s == 0) {     // nothing was computed; what has elements is zeros
        if (const int st = fill(ctx, dtype, dq, d->b, d->t, 2 * d->h, d->dh, p.dq); st != NOTT_OK) return st;
        if (const int st = fill(ctx, dtype, dk, d->b, d->s, 2 * d->hk, d->dh, p.dk); st != NOTT_OK) return st;
        if (const int st = fill(ctx, dtype, dv, d->b, d->s, d->hk, d->dv, p.dv_); st != NOTT_OK) return st;
        const int64_t one[3] = {0, 0, 1}, token[3] = {d->t * d->h, d->h, 1};
        if (d->token_lam) return fill(ctx, NOTT_F32, dlam, d->b, d->t, d->h, 1, token);
        return accumulate ? (int)NOTT_OK : fill(ctx, NOTT_F32, dlam, 1, 1, d->h, 1, one);
    }
    NOTT_REQUIRE(ctx, dO && q && k && v && lam && o && o2 && lse && dq && dk && dv && dlam, "nott_diff_attention_bwd: null buffer");
    p.lam = lam;
    p.lengths = lengths;
    p.start = q_start;
    const int elem = (int)nott::dtype_size(dtype);
    p.vec = even16(q, p.q, elem) && even16(k, p.k, elem) && even16(v, p.v, elem) && even16(dO, p.od, elem);
    const int64_t pairs = d->b * d->hk, total = pairs * p.rows;
    // Fewer key blocks than CUs: the rows are split, if the parts find room.  One workgroup a
    // CU with shares of 128 rows or more (3 x 105 tokens of 8 heads on 2, 128 + 256 columns 121
    // -> 84 us; 1024 tokens of 16 heads on 4, 279 -> 219, with two a CU 248; 256 tokens of 8
    // heads on 2, 64 + 128, 97 -> 48); causal blocks differ in length, and up to three for two CUs
    // even that out where shares keep 2048 rows (4096 tokens 1529 us with one, 1365 with 1.5,
    // 1416 with two).
    const bool fast = dtype == NOTT_BF16 && p.vec && p.dh % 8 == 0 && p.dv % 8 == 0 && even16(o, p.o, 2) && (uintptr_t)o2 % 16 == 0;
    const size_t stat_bytes = ((size_t)total * kStats * sizeof(float) + 255) & ~size_t(255);
    const int64_t key_blocks = pairs * ceil_div(p.s, mx::FIXED);
    float *stats = nullptr, *parts = nullptr;
    const int64_t one = std::min<int64_t>(ctx->num_cu / key_blocks, p.rows / 128);
    const int64_t n = p.causal ? std::max<int64_t>(one, std::min<int64_t>(ctx->num_cu * 3 / 2 / key_blocks, p.rows / 2048)) : one;
    if (fast && n > 1) {
        const size_t bytes = (size_t)n * pairs * p.s * (2 * p.dh + p.dv) * sizeof(float);
        if (char* ws = static_cast<char*>(nott::optional_workspace(ctx, stat_bytes + bytes))) {
            stats = reinterpret_cast<float*>(ws);
            parts = reinterpret_cast<float*>(ws + stat_bytes);
            p.nsplit = (int32_t)n;
        }
    }
    if (!stats) stats = static_cast<float*>(nott::workspace(ctx, stat_bytes));
    if (!stats) return NOTT_ERR_ALLOC;
    auto run = [&](auto type) {
        using T = decltype(type);
        const auto* tq = static_cast<const T*>(q);
        const auto* tk = static_cast<const T*>(k);
        const auto* tv = static_cast<const T*>(v);
        const auto* to = static_cast<const T*>(o);
        const auto* to2 = static_cast<const T*>(o2);
        const auto* tdo = static_cast<const T*>(dO);
        auto* tdq = static_cast<T*>(dq);
        auto* tdk = static_cast<T*>(dk);
        auto* tdv = static_cast<T*>(dv);
        if constexpr (sizeof(T) == 2) {
            if (fast) {
                return mx::with_blocks(p, [&](auto b, auto w) {
                    return mx::bwd<decltype(b)::value, decltype(w)::value>(ctx, p, pairs, tq, tk, tv, to, to2, tdo, lse, stats, parts,
                                                                           tdq, tdk, tdv, dlam);
                });
            }
        }
        switch (slices_for(p, AT<T>::SL)) {
            case 1: return any::bwd<T, 1>(ctx, p, pairs, tq, tk, tv, to, to2, tdo, lse, stats, tdq, tdk, tdv, dlam);
            case 2: return any::bwd<T, 2>(ctx, p, pairs, tq, tk, tv, to, to2, tdo, lse, stats, tdq, tdk, tdv, dlam);
            default: return any::bwd<T, 4>(ctx, p, pairs, tq, tk, tv, to, to2, tdo, lse, stats, tdq, tdk, tdv, dlam);
        }
    };
    const int st = dtype == NOTT_BF16 ? run(bf16_t()) : run(float());
    if (st != NOTT_OK || p.token_lam) return st;
    hipLaunchKernelGGL(diff_dlam_kernel, dim3((unsigned)d->h), dim3(1024), 0, ctx->stream, stats + 3 * total, dlam, d->b,
                       accumulate, p);
    return launch_status(ctx, "diff_dlam_kernel");
}
