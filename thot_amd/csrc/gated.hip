// Gated linear layer: [g | u] = x·wᵀ + b, h = act(g)·u, and its backward.
//
//   backward: dg = dh·u·act'(g), du = dh·act(g)
//             dx = [dg|du]·w, dw = [dg|du]ᵀ·x, db = Σ_rows [dg|du]
// h is rounded once from fp32 pre-activations.  In bf16 layers [dg|du] goes into the
// products as bf16 pieces cut toward zero: three for the fp32 dw (all 24 bits), two
// for dx, of which the second ends at 2^-15 of a value where dx itself is rounded to
// 2^-8 (one piece put as much into dx as its rounding: 2.3e-3 in the norm for 1.7e-3).
//
// fp32 layers take the bf16 matrix cores as well, wherever the products are large
// (products of bf16 pieces: Henry, Tang and Heinecke, Leveraging the bfloat16 Artificial
// Intelligence Datatype For Higher-Precision Computations, 2019):
// v = hi + mid + lo holds all 24 bits, and the six products of pieces that reach
// 2^-23 of the whole (hi·hi, hi·mid, mid·hi, mid·mid, hi·lo, lo·hi) are summed in
// fp32, the small ones first: six products, where the fp32 matrix instructions take
// the time of sixteen, and no further from 64 bits than those (8192 rows of 1024 ->
// 2048 395 to 411 us, 554 with fp32 instructions on tiles of the same engine; gradients
// 477 and 479 against 557 and 600).  A fourth piece is hi with 0 for an infinity or NaN: it
// takes hi's place in all products but hi·hi, so that an infinity enters a sum once, as
// its product.  The last piece ends at bf16's least number, so that values below 2^-110
// keep 2^-134 rather than their own last bit (inputs of 2^-110 come out with an error of
// 1.5e-7 in the norm as all others, of 2^-115 with 1.1e-6).
#include "gemm_dma.hpp"

namespace {

using namespace nott::gemm;
using nott::ceil_div;
using nott::launch_status;
using nott::WorkspaceHold;

// FAST (bf16 results): the exponent's rounding, |x|·2^-24 of the result, stays in;
// no clamp is needed then (exp2 ends in 0 or infinity, 1/infinity is 0).  Otherwise 0
// from where it would be below fp32's least normal number (x < −87.3).
template <bool FAST>
__device__ __forceinline__ float sigmoid(float x) {
    if constexpr (FAST) return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * -1.4426950f));
    const float e = exp_fine(__builtin_amdgcn_fmed3f(-x, -87.f, 87.3f));
    return x != x ? x : x < -87.3f ? 0.f : __builtin_amdgcn_rcpf(1.f + e);
}

// The activation (a) and its derivative (da).  g = ±infinity gives their limits: a
// product of g and a factor that ends in 0 takes −kLargest for −infinity, and the
// derivatives' terms take g within ±1e4, past which all of their exponentials are 0
// or 1 (a NaN stays in e or cdf).
constexpr float kLargest = 3.40282347e38f;
template <int ACT, bool FAST>
__device__ __forceinline__ void activate(float g, float& a, float& da) {
    const float from = fmaxf(g, -kLargest), near = __builtin_amdgcn_fmed3f(g, -1e4f, 1e4f);
    if constexpr (ACT == NOTT_ACT_SILU) {
        const float e = sigmoid<FAST>(g);
        a = from * e;
        da = fmaf(near * e, 1.f - e, e);
    } else if constexpr (ACT == NOTT_ACT_GELU) {
        const float cdf = 0.5f * erfcf(g * -0.70710678f);
        a = from * cdf;
        da = fmaf(near * 0.39894228f, exp_fine(fmaxf(-0.5f * near * near, -120.f)), cdf);
    } else if constexpr (ACT == NOTT_ACT_GELU_TANH) {
        const float e = sigmoid<FAST>(1.5957691f * fmaf(0.044715f * g, g * g, g));
        a = from * e;
        da = fmaf(near * e * (1.f - e), 1.5957691f * fmaf(0.134145f * near, near, 1.f), e);
    } else if constexpr (ACT == NOTT_ACT_RELU) {
        a = relu_out(g);
        da = g > 0.f ? 1.f : g != g ? g : 0.f;
    } else {
        a = sigmoid<FAST>(g);
        da = a * (1.f - a);
    }
}

template <class F>
__host__ __device__ __forceinline__ auto with_act(int act, F f) {
    switch (act) {
        case NOTT_ACT_SILU: return f(std::integral_constant<int, NOTT_ACT_SILU>());
        case NOTT_ACT_GELU: return f(std::integral_constant<int, NOTT_ACT_GELU>());
        case NOTT_ACT_GELU_TANH: return f(std::integral_constant<int, NOTT_ACT_GELU_TANH>());
        case NOTT_ACT_RELU: return f(std::integral_constant<int, NOTT_ACT_RELU>());
        default: return f(std::integral_constant<int, NOTT_ACT_SIGMOID>());
    }
}

// The forward's epilogue on the direct-to-LDS engine: a wave's TM×32 block of g
// and u (lane l: row l % 32, columns 8q + 4·(l/32) + e in register 4q + e of each
// 32×32 block) becomes h and, where asked for, [g | u], each staged through LDS as
// [row][32] and stored as whole row pieces of 64 (bf16) or 128 bytes.  bf16: the
// 16-byte chunk at chunk ^ (row/2 % 4), its halves exchanged on rows with bit 3
// set; fp32: at chunk ^ (row % 8).
// Bound by the matrix cores: 8192 rows of 1024 -> 4096 bf16 146 us (940 TFLOP/s, 300k
// cycles), 135 without [g | u]; a plain linear product of the same sizes 148 to 151.  After
// some 2 ms of such launches back to back each takes 172 to 190, the library's product
// 141 to 145 for 109: launches with pauses between them keep 146 and the same cycles.
template <typename T>
struct GatedStore {
    T* h;
    T* gu;
    const float* bias;
    int64_t m, f;
    int32_t act;
    bool vec;   // 16-byte stores fit every row
    static constexpr int E = 16 / (int)sizeof(T), C = 32 / E;   // a row's chunks
    static constexpr int kRowBytes = 32 * (int)sizeof(T);
    static __device__ __forceinline__ int at(int row, int chunk) {
        return row * kRowBytes + ((chunk ^ (sizeof(T) == 2 ? (row >> 1) & 3 : row & 7)) << 4);
    }
    // Columns 8q + 4·hf + 0..3 of a row.
    static __device__ __forceinline__ void put(char NOTT_LDS* buf, int row, int q, int hf, const float (&v)[4]) {
        if constexpr (sizeof(T) == 2) {
            const u32x2 w = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
            *reinterpret_cast<u32x2 NOTT_LDS*>(buf + at(row, q) + ((hf ^ ((row >> 3) & 1)) << 3)) = w;
        } else {
            *reinterpret_cast<f32x4 NOTT_LDS*>(buf + at(row, 2 * q + hf)) = f32x4{v[0], v[1], v[2], v[3]};
        }
    }
    template <int TM>
    __device__ __forceinline__ void flush(const char NOTT_LDS* buf, T* dst, int64_t ld, int64_t m0, int64_t c0,
                                          int lane) const {
        if (vec) {
            const int c = lane % C;
#pragma unroll
            for (int it = 0; it < TM * C / 64; ++it) {
                const int row = 64 / C * it + lane / C;
                u32x4 w = *reinterpret_cast<const u32x4 NOTT_LDS*>(buf + at(row, c));
                if (sizeof(T) == 2 && ((row >> 3) & 1)) w = u32x4{w.z, w.w, w.x, w.y};
                if (m0 + row < m && c0 + E * c < f) *reinterpret_cast<u32x4*>(dst + (m0 + row) * ld + c0 + E * c) = w;
            }
        } else {
            const int c = lane & 31;
            for (int it = 0; it < TM / 2; ++it) {
                const int row = 2 * it + (lane >> 5);
                const int b = sizeof(T) == 2 ? at(row, c >> 3) + ((((c >> 2) & 1) ^ ((row >> 3) & 1)) << 3) + (c & 3) * 2
                                             : at(row, c >> 2) + (c & 3) * 4;
                const T v = *reinterpret_cast<const T NOTT_LDS*>(buf + b);
                if (m0 + row < m && c0 + c < f) dst[(m0 + row) * ld + c0 + c] = v;
            }
        }
    }
    template <int TM, int FM>
    __device__ __forceinline__ void store_pair(f32x16 (&acc)[FM][2], char NOTT_LDS* buf, int64_t m0, int64_t c0,
                                               int lane) const {
        const int r = lane & 31, hf = lane >> 5;
        auto stage = [&](int which) {
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = acc[i][which][4 * q + e];
                    put(buf, 32 * i + r, q, hf, v);
                }
        };
        if (bias) {
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                float b[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int64_t c = c0 + 8 * (e >> 2) + 4 * hf + (e & 3);
                    b[e] = bias[(c < f ? c : f - 1) + w * f];
                }
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[i][w][e] += b[e];
            }
        }
        if (gu) {
            stage(0);
            flush<TM>(buf, gu, 2 * f, m0, c0, lane);
            stage(1);
            flush<TM>(buf, gu + f, 2 * f, m0, c0, lane);
        }
        with_act(act, [&](auto A) {
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float a, da;
                        activate<decltype(A)::value, sizeof(T) == 2>(acc[i][0][4 * q + e], a, da);
                        v[e] = a * acc[i][1][4 * q + e];
                    }
                    put(buf, 32 * i + r, q, hf, v);
                }
        });
        flush<TM>(buf, h, f, m0, c0, lane);
    }
};

// fp32, from bf16 pieces of x and w.
struct GatedPieces : GatedStore<float> {
    dma::Pieces pieces;
};

}  // namespace

template <> struct nott::gemm::dma::IsPaired<GatedStore<bf16_t>> { static constexpr bool value = true; };
template <> struct nott::gemm::dma::IsPaired<GatedPieces> { static constexpr bool value = true; };
template <> struct nott::gemm::dma::IsPieces<GatedPieces> { static constexpr bool value = true; };

namespace {

// h (and gu) from the fp32 products pre [m, 2f] and the bias.
template <int ACT>
__global__ __launch_bounds__(256) void gated_act_kernel(const float* __restrict__ pre, const float* __restrict__ b,
                                                        int64_t m, int64_t f, float* __restrict__ h,
                                                        float* __restrict__ gu) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= f) return;
    const float bg = b ? b[c] : 0.f, bu = b ? b[f + c] : 0.f;
    for (int64_t r = blockIdx.y; r < m; r += gridDim.y) {
        const float g = pre[r * 2 * f + c] + bg, u = pre[r * 2 * f + f + c] + bu;
        float a, da;
        activate<ACT, false>(g, a, da);
        h[r * f + c] = a * u;
        if (gu) {
            gu[r * 2 * f + c] = g;
            gu[r * 2 * f + f + c] = u;
        }
    }
}

// E fp32 values as bf16 (E = 1, 4 or 8; aligned to E elements).
template <int E>
__device__ __forceinline__ void store_piece(bf16_t* p, const float (&v)[E]) {
    if constexpr (E == 8) Pack16<bf16_t>::st(p, v);
    else if constexpr (E == 4) Vec4<bf16_t>::st(p, f32x4{v[0], v[1], v[2], v[3]});
    else *p = f32_to_bf16(v[0]);
}

// v (fp32 operands) as four bf16 pieces `stride` elements apart: the nearest, the nearest
// of what that leaves, of what both leave; and the first again with 0 in place of an
// infinity or NaN, which have nothing in the other two.  Finite values that round to an
// infinity take the largest finite piece.
constexpr int kPieces = 4;
template <int E>
__device__ __forceinline__ void store_nearest(bf16_t* out, int64_t stride, float (&v)[E]) {
    float hi[E], q[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const bool finite = fabsf(v[e]) <= kLargest;
        hi[e] = finite ? bf16_to_f32(f32_to_bf16(__builtin_amdgcn_fmed3f(v[e], -0x1.fep127f, 0x1.fep127f))) : 0.f;
        q[e] = finite ? hi[e] : v[e];
        v[e] = finite ? v[e] - hi[e] : 0.f;
    }
    store_piece<E>(out, q);
    store_piece<E>(out + 3 * stride, hi);
#pragma unroll
    for (int p = 1; p < 3; ++p) {
        store_piece<E>(out + p * stride, v);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] -= bf16_to_f32(f32_to_bf16(v[e]));
    }
}
// v cut to bf16 toward zero; NaN stays.
__device__ __forceinline__ float toward_zero(float v) {
    return v != v ? v : __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v) & 0xffff0000u);
}
// v as bf16 pieces `stride` elements apart, each cut toward zero from what the ones
// before leave; three hold all of its bits.  A value's pieces all have its sign and
// none is zero (2^-40 of the value, at least 2^-133, where nothing is left; an infinity
// again): so the sum of their products with an infinity is that infinity, as the
// value's own is, and not infinity − infinity or 0·infinity.
template <int E>
__device__ __forceinline__ void store_cut(bf16_t* out, int64_t stride, int pieces, float (&v)[E]) {
    float least[E];
#pragma unroll
    for (int e = 0; e < E; ++e)
        least[e] = v[e] == 0.f ? 0.f : __builtin_copysignf(fmaxf(fabsf(v[e]) * 0x1p-40f, 0x1p-133f), v[e]);
    for (int p = 0; p < pieces; ++p) {
        float q[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const bool none = v[e] == 0.f;
            q[e] = toward_zero(none ? least[e] : v[e]);
            if (!none && fabsf(v[e]) <= kLargest) v[e] -= q[e];
        }
        store_piece<E>(out + p * stride, q);
    }
}

// [dg|du] in rows of ld elements with zeros past 2f: as fp32 (whole, the generic
// engine's operand) and as bf16 pieces, each `stride` elements behind the one before:
// of a bf16 layer store_cut's, in fp32 store_nearest's.  A workgroup takes 64·E columns (E = 1, or
// whole 16-byte chunks where all rows fit them and ld is 2f) and every gridDim.y-th
// group of 4 rows; partial (null: no db) [gridDim.y][2f] receives its column sums of the unrounded
// values.  Bound by memory: 8192 x 4096 bf16 with three pieces, 604 MB, 96 us (6.3 TB/s;
// 108 in the mean of twenty calls in a row; two pieces an element at a time, 470 MB, 94).
template <typename T, int ACT, int E>
__global__ __launch_bounds__(256) void gated_dact_kernel(const T* __restrict__ dh, const T* __restrict__ gu, int64_t m,
                                                         int64_t f, int64_t ld, float* __restrict__ whole,
                                                         bf16_t* __restrict__ out, int pieces, int64_t stride,
                                                         float* __restrict__ partial) {
    __shared__ float red[2][4][64 * E];
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    const int64_t c = ((int64_t)blockIdx.x * 64 + lane) * E;
    float sg[E], su[E];
#pragma unroll
    for (int e = 0; e < E; ++e) sg[e] = su[e] = 0.f;
    auto load = [](const T* p, float (&v)[E]) {
        if constexpr (E == 1) v[0] = Io<T>::ld(p, 0);
        else Pack16<T>::ld(p, v);
    };
    auto store = [&](int64_t at, float (&v)[E]) {
        if (whole) {
#pragma unroll
            for (int e = 0; e < E; ++e) whole[at + e] = v[e];
        }
        if constexpr (sizeof(T) == 2) {
            store_cut<E>(out + at, stride, pieces, v);
        } else if (pieces) {
            store_nearest<E>(out + at, stride, v);
        }
    };
    if (c < f) {
        for (int64_t r = (int64_t)blockIdx.y * 4 + wid; r < m; r += (int64_t)gridDim.y * 4) {
            float g[E], u[E], d[E], dg[E], du[E];
            load(gu + r * 2 * f + c, g);
            load(gu + r * 2 * f + f + c, u);
            load(dh + r * f + c, d);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                float a, da;
                activate<ACT, sizeof(T) == 2>(g[e], a, da);
                dg[e] = d[e] * u[e] * da;
                du[e] = d[e] * a;
                sg[e] += dg[e];
                su[e] += du[e];
            }
            store(r * ld + c, dg);
            store(r * ld + f + c, du);
            if constexpr (E == 1) {
                for (int64_t j = 2 * f + c; j < ld; j += f) {
                    float none[1] = {0.f};
                    store(r * ld + j, none);
                }
            }
        }
    }
    if (!partial) return;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        red[0][wid][lane * E + e] = sg[e];
        red[1][wid][lane * E + e] = su[e];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * 64 * E; i += 256) {
        const int w = i / (64 * E), j = i % (64 * E);
        const int64_t col = (int64_t)blockIdx.x * 64 * E + j;
        if (col < f)
            partial[(int64_t)blockIdx.y * 2 * f + w * f + col] = (red[w][0][j] + red[w][1][j]) + (red[w][2][j] + red[w][3][j]);
    }
}

// db[c] (+)= Σ_z partial[z][c]: a workgroup has 64 columns, 16 threads of each taking
// every 16th slab, and adds their sums in order.
__global__ __launch_bounds__(1024) void gated_db_kernel(const float* __restrict__ partial, int slabs, int64_t n,
                                                        float* __restrict__ db, int accumulate) {
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, r = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + lane;
    red[r][lane] = c < n && r < slabs ? ordered_sum1(partial + r * n + c, 16 * n, (slabs - r + 15) / 16) : 0.f;
    __syncthreads();
    if (r != 0 || c >= n) return;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += red[i][lane];
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
// An epilogue, and split-K partials, for products of pieces.
template <class EP>
struct PiecesOf : EP {
    dma::Pieces pieces;
};
struct PiecesPartial : dma::PartialRowStore {
    dma::Pieces pieces;
};
__device__ __forceinline__ PiecesPartial at_split(const PiecesPartial& ep, int z) { return {ep.at(z), ep.pieces}; }

}  // namespace

template <class EP> struct nott::gemm::dma::IsPieces<PiecesOf<EP>> { static constexpr bool value = true; };
template <> struct nott::gemm::dma::IsBf16RowMajor<PiecesOf<RowMajorStore<bf16_t>>> { static constexpr bool value = true; };
template <> struct nott::gemm::dma::IsPieces<PiecesPartial> { static constexpr bool value = true; };

namespace {

// Rows of ld elements that all start on a 16-byte address.
template <typename T>
bool ok16(const T* p, int64_t ld) {
    return (uintptr_t)p % 16 == 0 && ld * (int64_t)sizeof(T) % 16 == 0;
}
// n rounded up to whole 16-byte chunks of bf16.
int64_t up8(int64_t n) { return (n + 7) & ~int64_t(7); }

// 16 bytes from any element's address.
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));

// src [rows, cols] to bf16 [prows, pcols] at dst, of fp32 store_nearest's pieces one behind
// the other, zeros past src's rows and columns.  No rows: nothing.
template <typename T>
struct PieceJob {
    const T* src = nullptr;
    int64_t rows = 0, cols = 0;
    bf16_t* dst = nullptr;
    int64_t chunks = 0;   // of 8 elements
    FastDiv row;          // chunks of a row
    PieceJob() = default;
    PieceJob(const T* s, int64_t r, int64_t c, bf16_t* d, int64_t prows, int64_t pcols)
        : src(s), rows(r), cols(c), dst(d), chunks(prows * pcols / 8), row((uint32_t)(pcols / 8)) {}
};
// Two jobs in one launch: the copy of a bf16 tensor whose rows no 16-byte load fits, and
// fp32 tensors for the bf16 engine.  A thread has 8 elements.
template <typename T>
__global__ __launch_bounds__(256) void pieces_kernel(PieceJob<T> a, PieceJob<T> b) {
    const PieceJob<T> j = blockIdx.y ? b : a;
    const bool small = j.chunks < (int64_t)1 << 32;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < j.chunks; i += (int64_t)gridDim.x * 256) {
        const int64_t r = small ? j.row.div((uint32_t)i) : i / j.row.d, c = (i - r * j.row.d) * 8;
        const T* p = j.src + r * j.cols + c;
        float v[8];
        if (r < j.rows && c + 8 <= j.cols) {
            if constexpr (sizeof(T) == 2) {
                const u32x4 raw = *reinterpret_cast<const u32x4_any*>(p);   // a copy: the reference would claim 16-byte alignment
                Pack16<bf16_t>::unpack(raw, v);
            } else {
                const f32x4 lo = reinterpret_cast<const f32x4_any*>(p)[0], hi = reinterpret_cast<const f32x4_any*>(p)[1];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = lo[e], v[4 + e] = hi[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = r < j.rows && c + e < j.cols ? Io<T>::ld(p, e) : 0.f;
        }
        if constexpr (sizeof(T) == 2) Pack16<bf16_t>::st(j.dst + i * 8, v);
        else store_nearest<8>(j.dst + i * 8, j.chunks * 8, v);
    }
}
template <typename T>
void to_pieces(nott_ctx ctx, const PieceJob<T>& a, const PieceJob<T>& b = {}) {
    const int64_t most = std::max(a.chunks, b.chunks);
    if (most == 0) return;
    const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(most, 256), 8192);
    hipLaunchKernelGGL(pieces_kernel<T>, dim3(blocks, b.chunks ? 2 : 1), dim3(256), 0, ctx->stream, a, b);
}

// Few rows (single tokens of some sequences): the weights are streamed once, 16
// gate rows and the matching 16 up rows a workgroup, its 8 waves dealing out 64
// k's at a time; x's rows are the other MFMA operand (16·MT of them), both straight
// from memory into registers in the operand layout (lane l: row l % 16, k =
// 8·(l/16) + 0..7 of each 32).  The waves' sums meet in LDS.  Rows may start at any
// address; TAIL: d >= 8 is no multiple of 8, and the last chunk of a row is the
// row's last 8 elements, moved down.
// 1 row of 1024 → 4096 4.9 us, 8 rows 5.4 (the 16.8 MB of weights take 3.4 at the
// copy rate), of 4096 → 11008 31 and 33 us.
template <int MT, bool TAIL>
__global__ __launch_bounds__(512) void gated_rows_kernel(const bf16_t* __restrict__ x, const bf16_t* __restrict__ w,
                                                         const float* __restrict__ bias, int64_t m, int64_t d, int64_t f,
                                                         int act, bf16_t* __restrict__ h, bf16_t* __restrict__ gu) {
    constexpr int NW = 8;
    __shared__ float red[NW][2][MT][256];
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    const int r = lane & 15, kq = lane >> 4;
    const int64_t c0 = (int64_t)blockIdx.x * 16;
    const int64_t row = c0 + r < f ? c0 + r : f - 1;
    const bf16_t* wg = w + row * d;
    const bf16_t* wu = wg + f * d;
    const bf16_t* xr[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) xr[t] = x + (16 * t + r < m ? 16 * t + r : m - 1) * d;
    auto chunk = [&](const bf16_t* p, int64_t k) {
        const int64_t at = k + 8 <= d ? k : d - 8;
        u32x4 v = *reinterpret_cast<const u32x4_any*>(p + at);
        if constexpr (TAIL) {
            unsigned __int128 b = __builtin_bit_cast(unsigned __int128, v);
            v = __builtin_bit_cast(u32x4, b >> (16 * ((int)(k - at) & 7)));
        }
        return k < d ? v : u32x4{0, 0, 0, 0};
    };
    f32x4 acc[2][MT];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    u32x4 g[2][2], u[2][2], b[2][2][MT];
    auto load = [&](int p, int64_t unit) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int64_t k = 64 * unit + 32 * s + 8 * kq;
            g[p][s] = chunk(wg, k);
            u[p][s] = chunk(wu, k);
#pragma unroll
            for (int t = 0; t < MT; ++t) b[p][s][t] = chunk(xr[t], k);
        }
    };
    auto mma = [&](int p) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const bf16x8 xv = __builtin_bit_cast(bf16x8, b[p][s][t]);
                acc[0][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, g[p][s]), xv, acc[0][t], 0, 0, 0);
                acc[1][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, u[p][s]), xv, acc[1][t], 0, 0, 0);
            }
    };
    const int64_t units = (d + 63) / 64;
    for (int64_t i = wid; i < units; i += 2 * NW) {   // two units of 64 k in flight
        load(0, i);
        const bool two = i + NW < units;
        if (two) load(1, i + NW);
        mma(0);
        if (two) mma(1);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int t = 0; t < MT; ++t) *reinterpret_cast<f32x4*>(&red[wid][i][t][lane * 4]) = acc[i][t];
    __syncthreads();
    // lane l's register e: token l % 16, column 4·(l/16) + e
    for (int p = threadIdx.x; p < MT * 256; p += 512) {
        const int c = p & 15, tok = p >> 4;
        const int at = ((c >> 2) * 16 + (tok & 15)) * 4 + (c & 3);
        const int64_t col = c0 + c;
        if (col >= f || tok >= m) continue;
        float g = bias ? bias[col] : 0.f, u = bias ? bias[f + col] : 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            g += red[i][0][tok >> 4][at];
            u += red[i][1][tok >> 4][at];
        }
        const float a = with_act(act, [&](auto A) {
            float a, da;
            activate<decltype(A)::value, true>(g, a, da);
            return a;
        });
        Io<bf16_t>::st(h, tok * f + col, a * u);
        if (gu) {
            Io<bf16_t>::st(gu, tok * 2 * f + col, g);
            Io<bf16_t>::st(gu, tok * 2 * f + f + col, u);
        }
    }
}

int forward_rows(nott_ctx ctx, int64_t m, int64_t d, int64_t f, int act, const bf16_t* x, const bf16_t* w,
                 const float* b, bf16_t* h, bf16_t* gu) {
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)ceil_div(f, 16)), dim3(512), 0, ctx->stream, x, w, b, m, d, f, act, h, gu);
    };
    const bool tail = d % 8 != 0;
    if (m <= 16) tail ? go(gated_rows_kernel<1, true>) : go(gated_rows_kernel<1, false>);
    else if (m <= 32) tail ? go(gated_rows_kernel<2, true>) : go(gated_rows_kernel<2, false>);
    else tail ? go(gated_rows_kernel<4, true>) : go(gated_rows_kernel<4, false>);
    return launch_status(ctx, "gated_linear");
}

// Whether gated_rows_kernel beats 128×128 tiles: it reads the weights at the copy
// rate for up to 16 rows and slower as x's operands join them, the tiles take
// 0.55 us for each 64 of d (and a copy of operands that lie badly).  1024 → 4096:
// 32 rows 7.1 us against 12.0, 64 rows 9.6 against 12.1; 4096 → 11008: 16 rows 37.0
// and 37.2, 32 rows 48 against 37, 64 rows 72 against 37.
bool takes_rows(nott_ctx ctx, int64_t m, int64_t d, int64_t f, bool padded) {
    if (m <= 16 || m > 64) return m <= 16;
    const double weights = 4.0 * (double)f * (double)d / 4.9e6;
    const double rounds = (double)ceil_div(ceil_div(f, 64), ctx->num_cu);
    return weights * (m <= 32 ? 1.35 : 2.0) <= rounds * (double)ceil_div(d, 64) * 0.55 + (padded ? 2 * weights + 2 : 0);
}

// C = A·B on the generic engine.
template <typename T, class LA, class LB, class EP>
int generic(nott_ctx ctx, const LA& la, const LB& lb, const EP& ep, int64_t M, int64_t N, int64_t K) {
    return small_grid(ctx, M, N) ? run_small<T>(ctx, la, lb, ep, M, N, K) : run<T>(ctx, la, lb, ep, M, N, K);
}
// The same of plain operands; AT, BT as in gemm_dma.hpp.
template <typename T, bool AT, bool BT, class EP>
int product(nott_ctx ctx, const T* A, int64_t lda, const T* B, int64_t ldb, const EP& ep, int64_t M, int64_t N,
            int64_t K) {
    auto vec = [](const T* p, int64_t ld) { return ((uintptr_t)p % 16) == 0 && (ld * (int64_t)sizeof(T)) % 16 == 0; };
    const RowKLoader<T> row_a{A, lda, M, K, vec(A, lda)};
    if constexpr (AT) return generic<T>(ctx, ColKLoader<T>{A, lda, M, K}, ColKLoader<T>{B, ldb, N, K}, ep, M, N, K);
    else if constexpr (BT) return generic<T>(ctx, row_a, ColKLoader<T>{B, ldb, N, K}, ep, M, N, K);
    else return generic<T>(ctx, row_a, RowKLoader<T>{B, ldb, N, K, vec(B, ldb)}, ep, M, N, K);
}
// Operands of the generic engine for products of pieces, one piece after the other along
// k.  R(row, k) = p[stride·(k / ld) + row·ld + k % ld] for two pieces of rows of ld
// elements, a multiple of 8: a chunk lies in one of them.
struct TwoPieces {
    static constexpr bool kRowFast = false;
    static constexpr int E = 8;
    const bf16_t* p;
    int64_t ld, rows, stride;
    __device__ __forceinline__ u32x4 chunk(int64_t row, int64_t k0) const {
        if (row >= rows || k0 >= 2 * ld) return u32x4{0, 0, 0, 0};
        return *reinterpret_cast<const u32x4*>(p + (k0 < ld ? 0 : stride - ld) + row * ld + k0);
    }
};
// R(row, k) = p[(k % period)·ld + row] for k < total, at most three periods; zero where
// k % period is K or more.
struct Repeated {
    static constexpr bool kRowFast = true;
    static constexpr int E = 8;
    const bf16_t* p;
    int64_t ld, rows, K, period, total;
    __device__ __forceinline__ u32x4 chunk(int64_t row, int64_t k0) const {
        bf16_t v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            int64_t k = k0 + e;
            if (k >= period) k -= period;
            if (k >= period) k -= period;
            v[e] = row < rows && k < K && k0 + e < total ? p[k * ld + row] : bf16_t(0);
        }
        return Pack<bf16_t>::make(v);
    }
};

// The six products of fp32 pieces (hi 0, mid 1, lo 2, finite hi 3), first factor and second:
// lo·hi, hi·lo, mid·mid, mid·hi, hi·mid, hi·hi.
constexpr uint32_t kPairs = 6, kFirst = 0x031132, kSecond = 0x013123;

// Whether an fp32 product of M×N×K, with so many elements to split into pieces, goes to
// the direct-to-LDS engine: its plan's time and the split's against the generic engine's
// 70 TFLOP/s, which spreads few tiles over the CUs by splitting k.  In us, generic and
// pieces (forward; dx and dw with the activation gradient): 1576 rows of 768 -> 2048 162
// and 87, 171 and 99, 140 and 103; 1024 of 768 -> 1024 42 and 57, 62 and 48, 58 and 48;
// 256 of 512 -> 1024 19 and 38, 22 and 29, 24 and 29.  On 25 sizes of 128 to 16384 rows
// the choice costs 1.4% over the better one in the mean (most where a forward of odd
// width has its loads element by element: 53 against 42).
bool takes_pieces(nott_ctx ctx, int64_t M, int64_t N, int64_t K, bool both_tr, bool split, int64_t elements) {
    const double us = dma::plan(ctx, M, N, kPairs * ceil_div(K, dma::BK) * dma::BK, both_tr, false, split ? 0 : 1).us;
    return us + 4 + (double)elements / 5e5 < 6 + 2.0 * (double)M * (double)N * (double)K / 70e6 &&
           ceil_div(M, 128) * ceil_div(N, 64) < (int64_t)1 << 23;
}

int fwd(nott_ctx ctx, int64_t m, int64_t d, int64_t f, int act, const bf16_t* x, const bf16_t* w, const float* b,
        bf16_t* h, bf16_t* gu) {
    const int64_t dp = up8(d);
    const bool rows = takes_rows(ctx, m, d, f, !ok16(w, d));
    if (rows && d >= 8) return forward_rows(ctx, m, d, f, act, x, w, b, h, gu);
    NOTT_REQUIRE(ctx, ceil_div(m, 128) * ceil_div(f, 64) < (int64_t)1 << 26, "nott_gated_linear_fwd: too large");
    const bool pad_x = !ok16(x, d), pad_w = !ok16(w, d);
    WorkspaceHold ws(ctx, sizeof(bf16_t) * (size_t)(((pad_x ? m : 0) + (pad_w ? 2 * f : 0)) * dp));
    if (ws.failed()) return NOTT_ERR_ALLOC;
    bf16_t* xp = reinterpret_cast<bf16_t*>(ws.p);
    bf16_t* wp = xp + (pad_x ? m * dp : 0);
    using Job = PieceJob<bf16_t>;
    to_pieces(ctx, pad_x ? Job(x, m, d, xp, m, dp) : Job(), pad_w ? Job(w, 2 * f, d, wp, 2 * f, dp) : Job());
    const bf16_t* X = pad_x ? xp : x;
    const bf16_t* W = pad_w ? wp : w;
    if (rows) return forward_rows(ctx, m, dp, f, act, X, W, b, h, gu);
    const GatedStore<bf16_t> ep{h, gu, b, m, f, act, ok16(h, f) && ok16(gu, f)};
    const dma::Plan p = dma::plan(ctx, m, 2 * f, dp, false, false, 1);
    return dma::launch_shape<false, false, false>(ctx, p.shape, X, dp, W, dp, ep, m, 2 * f, dp, 1, dp);
}

int fwd(nott_ctx ctx, int64_t m, int64_t d, int64_t f, int act, const float* x, const float* w, const float* b, float* h,
        float* gu) {
    const int64_t dp = up8(d);
    const size_t room = kPieces * sizeof(bf16_t) * (size_t)((m + 2 * f) * dp);
    if (!takes_pieces(ctx, m, 2 * f, dp, false, false, (m + 2 * f) * dp) || !nott::optional_workspace(ctx, room)) {
        WorkspaceHold ws(ctx, sizeof(float) * (size_t)(m * 2 * f));
        if (ws.failed()) return NOTT_ERR_ALLOC;
        float* pre = reinterpret_cast<float*>(ws.p);
        const RowMajorStore<float> ep{pre, 2 * f, m, 2 * f, nullptr};
        const int st = product<float, false, false>(ctx, x, d, w, d, ep, m, 2 * f, d);
        if (st != NOTT_OK) return st;
        with_act(act, [&](auto a) {
            hipLaunchKernelGGL((gated_act_kernel<decltype(a)::value>),
                               dim3((unsigned)ceil_div(f, 256), (unsigned)std::min<int64_t>(m, 65535)), dim3(256), 0,
                               ctx->stream, pre, b, m, f, h, gu);
        });
        return launch_status(ctx, "gated_linear");
    }
    WorkspaceHold ws(ctx, room);
    if (ws.failed()) return NOTT_ERR_ALLOC;
    bf16_t* xp = reinterpret_cast<bf16_t*>(ws.p);
    bf16_t* wp = xp + kPieces * m * dp;
    to_pieces(ctx, PieceJob<float>(x, m, d, xp, m, dp), PieceJob<float>(w, 2 * f, d, wp, 2 * f, dp));
    const int64_t deep = kPairs * ceil_div(dp, dma::BK) * dma::BK;
    const dma::Plan p = dma::plan(ctx, m, 2 * f, deep, false, false, 1);
    const GatedPieces ep{{h, gu, b, m, f, act, ok16(h, f) && ok16(gu, f)},
                         dma::pieces(kPairs, kFirst, kSecond, m * dp, 2 * f * dp, dp)};
    return dma::launch_shape<false, false, false>(ctx, p.shape, xp, dp, wp, dp, ep, m, 2 * f, dp, 1, deep);
}

constexpr int64_t kMostSums = 128;   // slabs of rows that each leave sums for db
// [dg|du] in rows of ld elements (zeros past 2·f), whole or as pieces (gated_dact_kernel); db.
template <typename T>
int activation_bwd(nott_ctx ctx, int64_t m, int64_t f, int64_t ld, int act, const T* dh, const T* gu, float* whole,
                   bf16_t* out, int pieces, float* db, int accumulate) {
    constexpr int E = 16 / (int)sizeof(T);
    const bool vec = ld == 2 * f && f >= 64 * E && ok16(dh, f) && ok16(gu, f);
    // about eight workgroups a CU, of at least 4 rows; fewer where each leaves sums for db
    const int64_t columns = ceil_div(f, 64 * (vec ? E : 1));
    const int64_t slabs = std::max<int64_t>(1, std::min<int64_t>({ceil_div(8 * (int64_t)ctx->num_cu, columns), ceil_div(m, 4),
                                                                  db ? kMostSums : 65535}));
    float* partial = nullptr;
    if (db) {
        partial = static_cast<float*>(nott::workspace(ctx, sizeof(float) * (size_t)(slabs * 2 * f)));
        if (!partial) return NOTT_ERR_ALLOC;
    }
    with_act(act, [&](auto a) {
        constexpr int A = decltype(a)::value;
        auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)columns, (unsigned)slabs), dim3(256), 0, ctx->stream, dh, gu, m, f, ld,
                               whole, out, pieces, m * ld, partial);
        };
        if (vec) go(gated_dact_kernel<T, A, E>);
        else go(gated_dact_kernel<T, A, 1>);
    });
    if (db)
        hipLaunchKernelGGL(gated_db_kernel, dim3((unsigned)ceil_div(2 * f, 64)), dim3(1024), 0, ctx->stream, partial,
                           (int)slabs, 2 * f, db, accumulate);
    return launch_status(ctx, "gated_linear backward");
}

// ep's M×N = Σ over the pairs of pieces, K deep each, rows and columns of A and B in
// whole chunks.
template <bool AT, bool BT, class EP>
int pieces_product(nott_ctx ctx, const bf16_t* A, int64_t lda, const bf16_t* B, int64_t ldb, const EP& ep,
                   const dma::Pieces& pc, int64_t M, int64_t N, int64_t K) {
    const int64_t deep = pc.count * ceil_div(K, dma::BK) * dma::BK;
    dma::Plan p = dma::plan(ctx, M, N, deep, AT && BT, false, 0);
    float* part = nullptr;
    if (p.splits > 1) {
        part = static_cast<float*>(nott::optional_workspace(ctx, sizeof(float) * (size_t)(p.splits * M * N)));
        if (!part) p = dma::plan(ctx, M, N, deep, AT && BT, false, 1);
    }
    if (!part)
        return dma::launch_shape<AT, BT, false>(ctx, p.shape, A, lda, B, ldb, PiecesOf<EP>{ep, pc}, M, N, K, 1, deep);
    const int st = dma::launch_shape<AT, BT, false>(ctx, p.shape, A, lda, B, ldb,
                                                    PiecesPartial{{part, nullptr, M, N}, pc}, M, N, K, p.splits, p.kps);
    if (st != NOTT_OK) return st;
    launch_splitk_reduce(ctx, part, p.splits, M, N, ep);
    return launch_status(ctx, "gated_linear splits");
}

int bwd(nott_ctx ctx, int64_t m, int64_t d, int64_t f, int act, const bf16_t* dh, const bf16_t* x, const bf16_t* w,
        const bf16_t* gu, bf16_t* dx, float* dw, float* db, int accumulate) {
    const int64_t dp = up8(d), fp = up8(2 * f);
    const int pieces = dw ? 3 : dx ? 2 : 0;
    // the direct-to-LDS engine, where a product has its 128 rows and columns
    const bool dma_dx = dx && m >= 128 && d >= 128, dma_dw = dw && 2 * f >= 128 && d >= 128;
    const bool pad_x = dma_dw && !ok16(x, d), pad_w = dma_dx && (!ok16(w, d) || fp != 2 * f);
    WorkspaceHold ws(ctx, sizeof(bf16_t) * (size_t)(m * fp * pieces + ((pad_x ? m : 0) + (pad_w ? fp : 0)) * dp));
    if (ws.failed()) return NOTT_ERR_ALLOC;
    bf16_t* dgu = reinterpret_cast<bf16_t*>(ws.p);
    bf16_t* xp = dgu + m * fp * pieces;
    bf16_t* wp = xp + (pad_x ? m * dp : 0);
    int st = activation_bwd(ctx, m, f, fp, act, dh, gu, nullptr, dgu, pieces, db, accumulate);
    if (st != NOTT_OK) return st;
    using Job = PieceJob<bf16_t>;
    to_pieces(ctx, pad_x ? Job(x, m, d, xp, m, dp) : Job(), pad_w ? Job(w, 2 * f, d, wp, fp, dp) : Job());
    if (dx) {   // the second piece, then the first
        const RowMajorStore<bf16_t> ep{dx, d, m, d, nullptr};
        st = dma_dx ? pieces_product<false, true>(ctx, dgu, fp, pad_w ? wp : w, dp, ep, dma::pieces(2, 0x01, 0x00, m * fp, 0, fp),
                                                  m, dp, fp)
                    : generic<bf16_t>(ctx, TwoPieces{dgu, fp, m, m * fp}, Repeated{w, d, d, 2 * f, fp, 2 * fp}, ep, m, d, 2 * fp);
        if (st != NOTT_OK) return st;
    }
    if (!dw) return st;
    const AccStore ep{dw, 2 * f, d, accumulate};
    if (!dma_dw)
        return generic<bf16_t>(ctx, ColKLoader<bf16_t>{dgu, fp, 2 * f, 3 * m}, Repeated{x, d, d, m, m, 3 * m}, ep, 2 * f, d,
                               3 * m);
    // third, second, first
    return pieces_product<true, true>(ctx, dgu, fp, pad_x ? xp : x, dp, ep, dma::pieces(3, 0x012, 0x000, m * fp, 0, m), fp, dp,
                                      m);
}

int bwd(nott_ctx ctx, int64_t m, int64_t d, int64_t f, int act, const float* dh, const float* x, const float* w,
        const float* gu, float* dx, float* dw, float* db, int accumulate) {
    const int64_t dp = up8(d), fp = up8(2 * f);
    bool pieces_dx = dx && takes_pieces(ctx, m, dp, fp, false, true, fp * dp);
    bool pieces_dw = dw && takes_pieces(ctx, fp, dp, m, true, true, m * dp);
    auto any = [&] { return pieces_dx || pieces_dw; };
    auto whole_too = [&] { return (dx && !pieces_dx) || (dw && !pieces_dw); };
    auto room = [&] {
        return sizeof(float) * (size_t)(whole_too() ? m * (any() ? fp : 2 * f) : 0) +
               kPieces * sizeof(bf16_t) * (size_t)((any() ? m * fp : 0) + ((pieces_dw ? m : 0) + (pieces_dx ? fp : 0)) * dp);
    };
    // no room for them and, behind them, db's sums: the generic engine
    if (any() && !nott::optional_workspace(ctx, room() + (db ? 256 + sizeof(float) * kMostSums * 2 * (size_t)f : 0)))
        pieces_dx = pieces_dw = false;
    const bool pieces = any(), whole = whole_too();
    const int64_t ld = pieces ? fp : 2 * f;
    WorkspaceHold ws(ctx, room());
    if (ws.failed()) return NOTT_ERR_ALLOC;
    bf16_t* dgu = reinterpret_cast<bf16_t*>(ws.p);
    bf16_t* xp = dgu + (pieces ? kPieces * m * fp : 0);
    bf16_t* wp = xp + (pieces_dw ? kPieces * m * dp : 0);
    float* all = reinterpret_cast<float*>(wp + (pieces_dx ? kPieces * fp * dp : 0));
    int st = activation_bwd(ctx, m, f, ld, act, dh, gu, whole ? all : nullptr, dgu, pieces ? kPieces : 0, db, accumulate);
    if (st != NOTT_OK) return st;
    using Job = PieceJob<float>;
    to_pieces(ctx, pieces_dx ? Job(w, 2 * f, d, wp, fp, dp) : Job(), pieces_dw ? Job(x, m, d, xp, m, dp) : Job());
    const AccStore to_dx{dx, m, d, 0}, to_dw{dw, 2 * f, d, accumulate};
    if (pieces_dx) {
        st = pieces_product<false, true>(ctx, dgu, fp, wp, dp, to_dx, dma::pieces(kPairs, kFirst, kSecond, m * fp, fp * dp, fp),
                                         m, dp, fp);
    } else if (dx) {
        st = product<float, false, true>(ctx, all, ld, w, d, to_dx, m, d, 2 * f);
    }
    if (st != NOTT_OK || !dw) return st;
    if (!pieces_dw) return product<float, true, true>(ctx, all, ld, x, d, to_dw, 2 * f, d, m);
    return pieces_product<true, true>(ctx, dgu, fp, xp, dp, to_dw, dma::pieces(kPairs, kFirst, kSecond, m * fp, m * dp, m), fp,
                                      dp, m);
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
        return fwd(ctx, m, d, f, act, static_cast<const float*>(x), static_cast<const float*>(w), b,
                          static_cast<float*>(h), static_cast<float*>(gu));
    return fwd(ctx, m, d, f, act, static_cast<const bf16_t*>(x), static_cast<const bf16_t*>(w), b,
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
        return bwd(ctx, m, d, f, act, static_cast<const float*>(dh), static_cast<const float*>(x),
                          static_cast<const float*>(w), static_cast<const float*>(gu), static_cast<float*>(dx), dw, db,
                          accumulate);
    return bwd(ctx, m, d, f, act, static_cast<const bf16_t*>(dh), static_cast<const bf16_t*>(x),
                       static_cast<const bf16_t*>(w), static_cast<const bf16_t*>(gu), static_cast<bf16_t*>(dx), dw, db,
                       accumulate);
}
