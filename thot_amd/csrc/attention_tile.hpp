// Tiles, fragments and MFMA forms that the attention kernels share (attention.hip: one
// softmax map a head; diff_attention.hip: two).
#pragma once

#include "lds_dma.hpp"

namespace nott {
namespace attn {

constexpr int kThreads = 256;     // 4 waves, 16 rows each
constexpr int BR = 64;            // rows per block (queries or keys)

template <typename T> struct AT;
template <> struct AT<float> { static constexpr int E = 4, SL = 16; };    // elems per 16 B, rows per 64-byte k-slice
template <> struct AT<bf16_t> { static constexpr int E = 8, SL = 32; };

// Tile of R rows × NCH 16-byte chunks: rows grouped by 16, chunk-major inside
// a group, slot XOR-swizzled by the chunk index (conflict-free for 16 lanes
// reading 16 rows of one chunk and for 16 lanes writing 16 chunks of a row).
__device__ __forceinline__ int toff(int row, int ch, int nch) {
    return (row >> 4) * (nch << 8) + (ch << 8) + (((row ^ ch) & 15) << 4);
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) { return pack_bf16x2(a, b); }

template <typename T>
__device__ __forceinline__ void mma(const u32x4& a, const u32x4& b, f32x4& acc) {
    if constexpr (sizeof(T) == 2) {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc,
                                                      0, 0, 0);
    } else {
        const f32x4 af = __builtin_bit_cast(f32x4, a), bf = __builtin_bit_cast(f32x4, b);
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(af.x, bf.x, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(af.y, bf.y, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(af.z, bf.z, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(af.w, bf.w, acc, 0, 0, 0);
    }
}

// Register tiles v[4] (4 × 16 k-slots) as MFMA A operands, packed once per
// block.  bf16: hi[s] is the 64-byte k-slice s rounded to bf16, tiles 2s and
// 2s+1 interleaved as k-slots {4q..4q+3, 16+4q..16+4q+3}; with LO, lo[s] is
// the bf16 remainder v − hi, so the two MFMAs carry ~16 mantissa bits (used
// for ds, whose entries are differences p∘(dp − rowsum) and lose the most to
// one bf16 rounding, and for p in the dk/dv pass).  fp32 passes the float
// vectors straight to the MFMA: building a u32x4 from bit-cast floats and
// casting it back makes hipcc (ROCm 7.2) feed the first component to all four
// v_mfma_f32_16x16x4_f32 issues.
template <typename T, bool LO>
struct RegA {
    u32x4 hi[2], lo[2];
    const f32x4* v;
    __device__ __forceinline__ explicit RegA(const f32x4 (&t)[4]) : v(t) {
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const f32x4 x = t[2 * s], y = t[2 * s + 1];
                hi[s] = u32x4{pack_bf16x2(x.x, x.y), pack_bf16x2(x.z, x.w), pack_bf16x2(y.x, y.y), pack_bf16x2(y.z, y.w)};
                if constexpr (LO) {
                    auto lo_of = [](uint32_t h, float a, float b) {
                        return pack_bf16x2(a - __builtin_bit_cast(float, h << 16),
                                           b - __builtin_bit_cast(float, h & 0xffff0000u));
                    };
                    lo[s] = u32x4{lo_of(hi[s].x, x.x, x.y), lo_of(hi[s].y, x.z, x.w), lo_of(hi[s].z, y.x, y.y),
                                  lo_of(hi[s].w, y.z, y.w)};
                }
            }
        }
    }
    // acc += A(slice s) · b
    __device__ __forceinline__ void mma(int s, const u32x4& b, f32x4& acc) const {
        if constexpr (sizeof(T) == 2) {
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, hi[s]), __builtin_bit_cast(bf16x8, b),
                                                          acc, 0, 0, 0);
            if constexpr (LO)
                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, lo[s]),
                                                              __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
        } else {
            const f32x4 af = v[s];
            const f32x4 bf = __builtin_bit_cast(f32x4, b);
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(af[0], bf[0], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(af[1], bf[1], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(af[2], bf[2], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(af[3], bf[3], acc, 0, 0, 0);
        }
    }
};

// Loads 16 bytes (E elements) of row `row` starting at column c0 of a
// [rows × dh] matrix, zero outside; vec = rows are 16-byte aligned.
template <typename T>
__device__ __forceinline__ u32x4 load_chunk(const T* base, int row, int nrows, int c0, int dh, int ld, bool vec) {
    constexpr int E = AT<T>::E;
    if (row >= nrows || c0 >= dh) return u32x4{0u, 0u, 0u, 0u};
    const T* p = base + (int64_t)row * ld + c0;
    if (vec && c0 + E <= dh) return *reinterpret_cast<const u32x4*>(p);
    T v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = (c0 + e < dh) ? p[e] : T(0);
    if constexpr (E == 8) {
        return u32x4{(uint32_t)v[0] | ((uint32_t)v[1] << 16), (uint32_t)v[2] | ((uint32_t)v[3] << 16),
                     (uint32_t)v[4] | ((uint32_t)v[5] << 16), (uint32_t)v[6] | ((uint32_t)v[7] << 16)};
    } else {
        return u32x4{__builtin_bit_cast(uint32_t, v[0]), __builtin_bit_cast(uint32_t, v[1]),
                     __builtin_bit_cast(uint32_t, v[2]), __builtin_bit_cast(uint32_t, v[3])};
    }
}

// Natural tile: rows r0..r0+63 of the matrix, [row][d], NCHD chunks per row.
template <typename T, int NCHD>
__device__ __forceinline__ void fill_nat(char* tile, const T* base, int r0, int nrows, int dh, int ld, bool vec) {
    constexpr int E = AT<T>::E;
    for (int t = threadIdx.x; t < BR * NCHD; t += kThreads) {
        const int ch = t % NCHD, row = t / NCHD;
        *reinterpret_cast<u32x4*>(tile + toff(row, ch, NCHD)) = load_chunk<T>(base, r0 + row, nrows, ch * E, dh, ld, vec);
    }
}

// A natural tile staged through registers, so that the next block's loads
// are in flight while the current block is computed: load() issues them,
// store() writes the tile after the barrier.  With 16-byte aligned rows and
// dh a multiple of the chunk width, every load is unconditional (rows past
// the end re-read a valid row and are zeroed at the store).
template <typename T, int NCHD>
struct TileRegs {
    static constexpr int E = AT<T>::E;
    static constexpr int N = (BR * NCHD + kThreads - 1) / kThreads;
    u32x4 r[N];
    uint32_t ok = 0;
    __device__ __forceinline__ void load(const T* base, int r0, int nrows, int dh, int ld, bool vec) {
        if (vec && dh % E == 0) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int t = threadIdx.x + j * kThreads;
                const int ch = t % NCHD, row = r0 + t / NCHD;
                const bool good = t < BR * NCHD && row < nrows && ch * E < dh;
                const int rr = row < nrows ? row : nrows - 1;
                r[j] = *reinterpret_cast<const u32x4*>(base + (int64_t)rr * ld + (ch * E < dh ? ch * E : 0));
                ok = good ? (ok | (1u << j)) : (ok & ~(1u << j));
            }
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int t = threadIdx.x + j * kThreads;
                const int ch = t % NCHD, row = t / NCHD;
                r[j] = t < BR * NCHD ? load_chunk<T>(base, r0 + row, nrows, ch * E, dh, ld, vec) : u32x4{0u, 0u, 0u, 0u};
            }
            ok = ~0u;
        }
    }
    __device__ __forceinline__ void store(char* tile) const {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int t = threadIdx.x + j * kThreads;
            if (t < BR * NCHD)
                *reinterpret_cast<u32x4*>(tile + toff(t / NCHD, t % NCHD, NCHD)) =
                    (ok >> j) & 1u ? r[j] : u32x4{0u, 0u, 0u, 0u};
        }
    }
};

// Row (within a 64-row block) stored at k-slot position `pos` of the
// transposed tile (the bf16 interleave described above; identity for fp32).
template <typename T>
__device__ __forceinline__ int perm_row(int pos) {
    if constexpr (sizeof(T) == 2) {
        const int s = pos >> 5, w = pos & 31, q = w >> 3, j = w & 7;
        return (s << 5) + (j < 4 ? 4 * q + j : 16 + 4 * q + (j - 4));
    } else {
        return pos;
    }
}

// Transposed tile: [d][row-position] for rows r0..r0+63, NCHT = 64·sizeof(T)/16
// chunks per d-row; DP rows (padded head dim).  One task moves an E×E block:
// E rows (at E consecutive positions) × E columns, transposed in registers.
template <typename T, int DP>
__device__ __forceinline__ void fill_trans(char* tile, const T* base, int r0, int nrows, int dh, int ld, bool vec) {
    constexpr int E = AT<T>::E;
    constexpr int NCHT = BR / E;
    constexpr int TASKS = NCHT * (DP / E);
    for (int t = threadIdx.x; t < TASKS; t += kThreads) {
        const int pc = t % NCHT, dc = t / NCHT;     // position chunk, d chunk
        u32x4 in[E], out[E];
#pragma unroll
        for (int i = 0; i < E; ++i) in[i] = load_chunk<T>(base, r0 + perm_row<T>(pc * E + i), nrows, dc * E, dh, ld, vec);
        if constexpr (E == 8) {
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t a = in[2 * e][d], b = in[2 * e + 1][d];
                    out[2 * d][e] = (a & 0xffffu) | (b << 16);
                    out[2 * d + 1][e] = (a >> 16) | (b & 0xffff0000u);
                }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) out[j] = u32x4{in[0][j], in[1][j], in[2][j], in[3][j]};
        }
#pragma unroll
        for (int i = 0; i < E; ++i) *reinterpret_cast<u32x4*>(tile + toff(dc * E + i, pc, NCHT)) = out[i];
    }
}

// Fragment of 16 rows (r0..r0+15) of a natural/transposed tile at 64-byte k-slice s.
__device__ __forceinline__ u32x4 frag(const char* tile, int r0, int s, int nch) {
    const int lane = threadIdx.x & 63;
    return *reinterpret_cast<const u32x4*>(tile + toff(r0 + (lane & 15), 4 * s + (lane >> 4), nch));
}

typedef short v4i16 __attribute__((ext_vector_type(4)));

// bf16 B fragment for columns d0..d0+15 whose 8 k-slots are rows ra+0..3 and
// rb+0..3 of a natural [row][d] tile (ra, rb per 16-lane group), read with
// two transposing LDS reads (ds_read_b64_tr_b16: within each 16-lane group,
// result lane j, element e comes from lane 4e + j/4, element j % 4; so lane
// s reads the 4 columns d0 + 4·(s%4).. of row ra + s/4).
__device__ __forceinline__ u32x4 frag_tr(const char* tile, int nch, int ra, int rb, int d0) {
    const int s = threadIdx.x & 15;
    const int d = d0 + 4 * (s & 3);
    const int ch = d >> 3, byte = (d & 7) * 2;
    const v4i16 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) v4i16*)(tile + toff(ra + (s >> 2), ch, nch) + byte));
    const v4i16 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) v4i16*)(tile + toff(rb + (s >> 2), ch, nch) + byte));
    const u32x2 xu = __builtin_bit_cast(u32x2, x), yu = __builtin_bit_cast(u32x2, y);
    return u32x4{xu.x, xu.y, yu.x, yu.y};
}

// B operand of the second-stage MFMAs (p·v, pᵀ·do, dsᵀ·q, ds·k): columns
// d0 = 16·dt, k-slice s of the register-resident tiles.  bf16 reads the
// natural tile with transposing reads, in the key interleave of RegA
// (k-slots 0..3 = rows 32s + 4·kq + e, 4..7 = rows 32s + 16 + 4·kq + e); fp32
// reads the transposed tile.
template <typename T, int NCHD, int NCHT>
__device__ __forceinline__ u32x4 frag2(const char* nat, const char* trans, int dt, int s) {
    if constexpr (sizeof(T) == 2) {
        const int kq = (threadIdx.x & 63) >> 4;
        return frag_tr(nat, NCHD, 32 * s + 4 * kq, 32 * s + 16 + 4 * kq, dt * 16);
    } else {
        return frag(trans, dt * 16, s, NCHT);
    }
}

// bf16 on 32×32×16 MFMAs: tiles of whole 64-byte column blocks, filled by direct-to-LDS loads.
namespace mx32 {

using lds::barrier;
using lds::dma16;
using lds::dma4;
using lds::lds_addr;
using lds::wait_vm_lgkm0;

constexpr int NW = 4;                    // waves per workgroup, 32 fixed rows each
constexpr int FIXED = 32 * NW;           // fixed rows per workgroup

static __device__ u32x4 zero_chunk;      // source of the padding columns

// Where chunk c of row r sits in its row.  In 256 bytes of banks a row of 4·ND
// chunks starts at chunk 4·ND·r mod 16; what is left of r's low 4 bits is
// XORed in: all of a 16-chunk row's, 2 bits of a 4- or 12-chunk one's.
template <int ND>
__device__ __forceinline__ int swz(int r, int c) {
    if constexpr (ND % 4 == 0) return c ^ (((r & 3) << 2) | ((r >> 2) & 3));
    else if constexpr (ND % 4 == 2) return c ^ ((r >> 1) & 7);
    else return c ^ ((r >> 2) & 3);
}
template <int ND>
__device__ __forceinline__ int tile_off(int r, int c) { return r * (64 * ND) + (swz<ND>(r, c) << 4); }

// Fills a [ROWS][32·ND] tile with rows row0.. of `base` (row stride ld, rows
// past nrows clamped to the last): 1 KB blocks dealt to the waves.  WHOLE: dh is
// 32·ND, so no chunk is padding.
template <int ND, int ROWS, bool WHOLE = false>
__device__ __forceinline__ void fill_tile(const bf16_t* base, int row0, int nrows, int dh, int ld, char NOTT_LDS* tile,
                                          int wid, int lane) {
    constexpr int CH = 4 * ND, BLOCKS = ROWS * CH / 64;
    static_assert(BLOCKS % NW == 0, "blocks split evenly over the waves");
#pragma unroll
    for (int qq = 0; qq < BLOCKS / NW; ++qq) {
        const int q = wid + NW * qq;
        const int i = 64 * q + lane, r = i / CH;
        const int c = swz<ND>(r, i - r * CH);   // (an involution)
        const int gr = min(row0 + r, nrows - 1);
        const bf16_t* src = base + (int64_t)gr * ld + 8 * c;
        dma16(WHOLE || 8 * c < dh ? src : reinterpret_cast<const bf16_t*>(&zero_chunk), lds_addr(tile) + 1024 * q);
    }
}

// 32×16 operand of tile rows r0..r0+31, d slice s: lane l gets row r0 + l%32,
// d = 16s + 8·(l/32) + 0..7.
template <int ND>
__device__ __forceinline__ bf16x8 frag_rows(const char NOTT_LDS* tile, int r0, int s, int lane) {
    return __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4 NOTT_LDS*>(
                                          tile + tile_off<ND>(r0 + (lane & 31), 2 * s + (lane >> 5))));
}

typedef short v4i16s __attribute__((ext_vector_type(4)));

// 32×16 operand of the transposed tile over the 16 rows from rs: lane l gets
// column d0 + l%32 and, as its 8 k-slots, rows rs + 4h + 0..3, rs + 8 + 4h +
// 0..3 (h = l/32): the rows that 8 consecutive registers of a 32×32
// accumulator hold, so a score tile is the other operand as it is.
template <int ND>
__device__ __forceinline__ bf16x8 frag_cols(const char NOTT_LDS* tile, int rs, int d0, int lane) {
    const int j = lane & 15, g = lane >> 4;
    const int col = d0 + 16 * (g & 1) + 4 * (j & 3);
    const int r1 = rs + 4 * (g >> 1) + (j >> 2);
    const int byte = (col & 7) * 2;
    const v4i16s lo =
        __builtin_amdgcn_ds_read_tr16_b64_v4i16((v4i16s NOTT_LDS*)(tile + tile_off<ND>(r1, col >> 3) + byte));
    const v4i16s hi =
        __builtin_amdgcn_ds_read_tr16_b64_v4i16((v4i16s NOTT_LDS*)(tile + tile_off<ND>(r1 + 8, col >> 3) + byte));
    const v4i16s w[2] = {lo, hi};
    return __builtin_bit_cast(bf16x8, w);
}

// Registers base..base+7 of an accumulator tile as a bf16 operand.
__device__ __forceinline__ bf16x8 pack8(const f32x16& t, int base) {
    const u32x4 w = {pack_bf16x2(t[base], t[base + 1]), pack_bf16x2(t[base + 2], t[base + 3]),
                     pack_bf16x2(t[base + 4], t[base + 5]), pack_bf16x2(t[base + 6], t[base + 7])};
    return __builtin_bit_cast(bf16x8, w);
}

// The remainder x − bf16(x) of registers base..base+7, rounded to bf16.
__device__ __forceinline__ bf16x8 pack8_lo(const f32x16& t, int base, const bf16x8& hi) {
    const u32x4 h = __builtin_bit_cast(u32x4, hi);
    auto lo2 = [&](int i, uint32_t w) {
        return pack_bf16x2(t[base + i] - __builtin_bit_cast(float, w << 16),
                           t[base + i + 1] - __builtin_bit_cast(float, w & 0xffff0000u));
    };
    const u32x4 w = {lo2(0, h.x), lo2(2, h.y), lo2(4, h.z), lo2(6, h.w)};
    return __builtin_bit_cast(bf16x8, w);
}

__device__ __forceinline__ f32x16 mfma(const bf16x8& a, const bf16x8& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// Maximum over lanes l and l ^ 32 (permlane32_swap of a value with itself gives
// the lower and the upper half's in every lane).
__device__ __forceinline__ float max_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x),
                                                    false, false);
    // through scalars: a bit-cast of a vector's element 1 reads element 0 (hipcc, ROCm 7.2)
    const unsigned lo = r[0], hi = r[1];
    return fmaxf(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
}

// A row's values as 2·ND B-operand slices: lane l holds d = 16s + 8·(l/32) + 0..7.
template <int ND, bool WHOLE = false>
__device__ __forceinline__ void load_fixed(const bf16_t* base, int row, int nrows, int dh, int ld, int lane,
                                           u32x4 (&r)[2 * ND]) {
    const bf16_t* pr = base + (int64_t)min(row, nrows - 1) * ld;
#pragma unroll
    for (int s = 0; s < 2 * ND; ++s) {
        const int d = 16 * s + 8 * (lane >> 5);
        r[s] = *reinterpret_cast<const u32x4*>(pr + (WHOLE || d < dh ? d : 0));
        if (!WHOLE && d >= dh) r[s] = u32x4{0u, 0u, 0u, 0u};
    }
}

}  // namespace mx32
}  // namespace attn
}  // namespace nott
