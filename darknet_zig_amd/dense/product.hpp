// product.hpp -- bf16 matrix products with an epilogue, fp32 sums:
//     out(r, c) = epilogue(sum over k of v(r, k) * u(c, k)).
//
// An operand is k-contiguous (element (row, k) at p[row * ld + k]) or
// row-contiguous (at p[k * ld + row]). v_mfma_f32_32x32x16_bf16 takes u as its
// A operand, so that a lane holds four consecutive columns c of one row r in
// consecutive registers: the epilogues store four at a time.
//
// A workgroup owns BR rows x BC columns, its waves WR x WC parts of that. K
// advances in slabs of BK = 64. In LDS a k-contiguous operand's slab is [row][64
// k], a lane's operand (eight k of its row) one 128-bit read; a row-contiguous
// one is [k][rows], read transposed (ds_read_b64_tr_b16: sixteen lanes take a
// block of four k and sixteen rows, each lane the four k of one row). The
// 16-byte chunks of a line are permuted so that what is read together lies in
// different banks (64 of four bytes: sixteen rows of 128 bytes two by two, four
// lines of k): no conflicts, where chunk ^ (row & 7) had four extra cycles a read
// (4096^3 118 us, 115.5 without).
//
// At 4096^3 the 256x256 tiles take 108 us (1270 TFLOP/s; 1320 and 1390 with one
// and both operands row-contiguous), at 8192^3 856 us (1284), where the library's
// products reach 1410, 1340 and 1160 (8192x16384x4096, both k-contiguous: 942 us here
// with a bias, 709 the library's). The matrix cores are busy 72% of the
// cycles, at the 1.9 GHz that the card holds under this load.
#pragma once

#include "dense_internal.hpp"

namespace dkz {
namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef short s16x8u __attribute__((ext_vector_type(8), aligned(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// The 16-byte chunk that slot `slot` of line `line` of a slab in LDS holds, and
// the other way round. A line is a row's 64 k, or (MC) one k's R rows.
template <int R, int BK, bool MC>
__device__ __forceinline__ uint32_t permuted(uint32_t line, uint32_t slot) {
    static_assert(BK == 64, "eight chunks a row");
    return MC ? slot ^ ((line & 3) * 4 & (R / 8 - 1)) : slot ^ (line >> 1 & 7);
}

struct ProductArgs {
    const __bf16 *v, *u;  // row side, column side
    uint32_t ldv, ldu;
    uint32_t rows, cols, k;
    uint32_t tiles_r, tiles_c, splits, k_chunk;  // k_chunk: a split's K, a multiple of the slab's depth
    float *partial;                              // splits > 1: [splits][rows][ldp]
    uint32_t ldp;
    uint32_t first_block;  // the launch's first workgroup among the product's
};

// A product's columns are u's rows, or (kPaired of its epilogue) come in eights of two
// halves in turn, each of `half` rows of u: columns 16 * i + 0 .. 7 are rows 8 * i + 0 .. 7
// and columns 16 * i + 8 .. 15 the same of the other half, so that a lane that has
// sixteen columns has eight pairs. Column `c` is there if unit(c) < half.
template <class Epi>
constexpr bool kPaired = false;
struct Pairs {
    static __device__ __forceinline__ uint32_t unit(uint32_t c) { return c / 16 * 8 + c % 8; }
    static __device__ __forceinline__ uint32_t row(uint32_t c, uint32_t half) { return (c / 8 & 1) * half + unit(c); }
};

// Consecutive workgroups go round the 8 XCDs: gives each XCD a run of neighbours.
__device__ __forceinline__ uint32_t xcd_run(uint32_t w, uint32_t total) {
    const uint32_t x = w & 7, q = total >> 3, rem = total & 7;
    return x * q + min(x, rem) + (w >> 3);
}

// Tile t's row and column of tiles: groups of eight tile rows, column by column.
__device__ __forceinline__ void tile_of(uint32_t t, uint32_t tiles_r, uint32_t tiles_c, uint32_t &tr, uint32_t &tc) {
    const uint32_t per_group = 8 * tiles_c, first = t / per_group * 8;
    const uint32_t in_group = t % per_group, size = min(tiles_r - first, 8u);
    tr = first + in_group % size;
    tc = in_group / size;
}

// Eight elements at any alignment of theirs: the whole words that hold them,
// shifted (a 16-byte load at an odd element is taken apart by the hardware).
__device__ __forceinline__ s16x8 load_shifted(const short *p) {
    const uint32_t *q = reinterpret_cast<const uint32_t *>((uintptr_t)p & ~(uintptr_t)3);
    const uint32_t odd = (uint32_t)(uintptr_t)p >> 1 & 1;
    const u32x4u x = *reinterpret_cast<const u32x4u *>(q);
    const uint32_t end = q[3 + odd];
    const u32x4 y = {__builtin_amdgcn_alignbit(x.y, x.x, 16 * odd), __builtin_amdgcn_alignbit(x.z, x.y, 16 * odd),
                     __builtin_amdgcn_alignbit(x.w, x.z, 16 * odd), __builtin_amdgcn_alignbit(end, x.w, 16 * odd)};
    return __builtin_bit_cast(s16x8, y);
}

// A slab of R rows of an operand on its way to LDS through registers, whatever
// its alignment. MC: row-contiguous.
template <int R, int BK, bool MC, int THREADS>
struct Staged {
    static constexpr int kChunks = R * BK / 8 / THREADS, kLine = MC ? R / 8 : BK / 8;  // kLine: chunks a line
    static_assert(kChunks * 8 * THREADS == R * BK, "whole chunks a thread");
    s16x8 v[kChunks];

    // Rows past `rows` and k past `kend` read as 0. A chunk that ends past its
    // line's end is the line's last eight elements, shifted: no branches but the
    // workgroup's, so that a thread's loads are all on their way at once.
    __device__ __forceinline__ void load(const __bf16 *p, uint32_t ld, uint32_t r0, uint32_t rows, uint32_t k0, uint32_t kend) {
        const short *base = reinterpret_cast<const short *>(p);
        const bool inside = r0 + R <= rows && k0 + BK <= kend;
        const uint32_t length = MC ? rows : kend, lines = MC ? kend : rows;
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const uint32_t c = threadIdx.x + i * THREADS;
            const uint32_t along = (MC ? r0 : k0) + c % kLine * 8, line = (MC ? k0 : r0) + c / kLine;
            if (inside) {
                v[i] = *reinterpret_cast<const s16x8u *>(base + (uint64_t)line * ld + along);
            } else if (length >= 8) {
                const uint32_t from = min(along, length - 8), shift = along - from;
                const s16x8 x = *reinterpret_cast<const s16x8u *>(base + (uint64_t)min(line, lines - 1) * ld + from);
                const u64x2 w = __builtin_bit_cast(u64x2, x);
                const uint64_t lo = shift & 4 ? w.y : w.x, hi = shift & 4 ? 0 : w.y;
                const uint32_t bits = (shift & 3) * 16;
                const bool none = shift >= 8 || line >= lines;
                const u64x2 y = {none ? 0 : lo >> bits | hi << 1 << (63 - bits), none ? 0 : hi >> bits};
                v[i] = __builtin_bit_cast(s16x8, y);
            } else {
                s16x8 x = {};
#pragma unroll
                for (int j = 0; j < 7; ++j)
                    if (line < lines && along + j < length) x[j] = base[(uint64_t)line * ld + along + j];
                v[i] = x;
            }
        }
    }
    // The same for columns r0 .. r0 + R - 1 in pairs.
    __device__ __forceinline__ void load_pairs(const __bf16 *p, uint32_t ld, uint32_t r0, uint32_t half, uint32_t k0, uint32_t kend) {
        static_assert(!MC, "rows of u with k contiguous");
        const short *base = reinterpret_cast<const short *>(p);
        const bool inside = r0 + R <= 2 * half && k0 + BK <= kend;
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const uint32_t c = threadIdx.x + i * THREADS, along = k0 + c % kLine * 8, col = r0 + c / kLine;
            const short *line = base + (uint64_t)min(Pairs::row(col, half), 2 * half - 1) * ld;
            if (inside) {
                v[i] = *reinterpret_cast<const s16x8u *>(line + along);
            } else {
                s16x8 x = {};
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (Pairs::unit(col) < half && along + j < kend) x[j] = line[along + j];
                v[i] = x;
            }
        }
    }
    __device__ __forceinline__ void store(char *lds) const {
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const uint32_t c = threadIdx.x + i * THREADS;
            const uint32_t line = c / kLine;
            *reinterpret_cast<s16x8 *>(lds + (line * kLine + permuted<R, BK, MC>(line, c % kLine)) * 16) = v[i];
        }
    }
};

// Rows row .. row + 31 of a slab in LDS, k 16 * step + 8 * (lane / 32) + 0 .. 7, as an MFMA operand.
template <int R, int BK, bool MC>
__device__ __forceinline__ bf16x8 fragment(const char *lds, uint32_t row, int step) {
    const uint32_t lane = threadIdx.x & 63;
    if constexpr (!MC) {
        const uint32_t r = row + (lane & 31), chunk = 2 * step + (lane >> 5);
        return *reinterpret_cast<const bf16x8 *>(lds + r * (BK * 2) + permuted<R, BK, MC>(r, chunk) * 16);
    } else {
        // Lane a of a group of sixteen names four rows of k line a / 4.
        const uint32_t a = lane & 15, k = 16 * step + 8 * (lane >> 5) + a / 4, r = row + (lane & 16) + 4 * (a & 3);
        const uint32_t at = k * (R * 2) + permuted<R, BK, MC>(k, r >> 3) * 16 + (r & 4) * 2;
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(lds + at));
        const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(lds + at + 4 * R * 2));
        const s16x8 both = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
        return __builtin_bit_cast(bf16x8, both);
    }
}

// A slab of R rows of an operand on its way straight to LDS (buffer loads with
// the lds bit: a wave's 64 lanes fill 1024 consecutive bytes, so the chunk
// permutation is applied to the addresses read). For operands whose rows lie on
// 16-byte boundaries. Chunks past `rows` or `kend` read past the buffer's end,
// which gives zeros.
template <int R, int BK, bool MC, int THREADS>
struct Direct {
    static constexpr int kLoads = R * BK / 8 / THREADS, kLine = MC ? R / 8 : BK / 8;
    static_assert(kLoads * 8 * THREADS == R * BK, "whole loads a thread");
    static constexpr uint32_t kOutside = 0x80000000u;
    uint32_t off[kLoads];  // bytes from the slab's first element; kOutside: past the rows
    uint32_t k[kLoads];    // the chunk's first k in the slab

    __device__ __forceinline__ void init(uint32_t ld, uint32_t r0, uint32_t rows) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const uint32_t c = threadIdx.x + i * THREADS;
            const uint32_t line = c / kLine, chunk = permuted<R, BK, MC>(line, c % kLine);
            k[i] = MC ? line : chunk * 8;
            off[i] = r0 + (MC ? chunk * 8 : line) < rows ? (line * ld + chunk * 8) * 2 : kOutside;
        }
    }
    // The same for columns r0 .. r0 + R - 1 in pairs; p is row r0 / 2.
    __device__ __forceinline__ void init_pairs(uint32_t ld, uint32_t r0, uint32_t half) {
        static_assert(!MC && R % 16 == 0, "rows of u with k contiguous");
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const uint32_t c = threadIdx.x + i * THREADS;
            const uint32_t line = c / kLine, chunk = permuted<R, BK, MC>(line, c % kLine);
            k[i] = chunk * 8;
            off[i] = Pairs::unit(r0 + line) < half ? (Pairs::row(line, half) * ld + chunk * 8) * 2 : kOutside;
        }
    }
    // Load i of a slab to LDS address `to` (the slab's). p: element (r0, k0);
    // left: k from k0 to the end, 0 past it. In asm, so that the compiler does
    // not make every later read of LDS wait for it: the loop below waits itself
    // (await_loads). (The address in LDS is in m0, which the load may read two wait
    // states after. Scalars that a vector instruction wrote would need five, which
    // cost 0.5% in every load; in the code as it is built there are none, and a test
    // looks.)
    __device__ __forceinline__ void load(int i, const __bf16 *p, uint32_t left, uint32_t to) const {
        const uint64_t at = (uint64_t)p;
        const i32x4 buf = {(int)(uint32_t)at, (int)(uint32_t)(at >> 32), (int)kOutside, 0x00020000};
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                     :
                     : "s"(to + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 1024 + i * THREADS * 16),
                       "v"(k[i] < left ? off[i] : kOutside), "s"(buf)
                     : "m0");
    }
};

// Waits for this wave's reads of LDS and all but its last N loads to it, then for the workgroup's other waves.
template <int N>
__device__ __forceinline__ void await_loads() {
    static_assert(N < 64, "the counter has six bits");
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// A wave's block of 32 rows, j of its part, to LDS: a row's chunk of four columns
// at chunk ^ row. (The writes of every block are there once, behind a branch on j,
// which is the same in all lanes.)
template <int TR, int TC>
__device__ __forceinline__ void block_to_lds(const f32x16 (&acc)[TC][TR], int j, float4 *part) {
    constexpr uint32_t kChunks = TC * 8, kMask = kChunks - 1;
    const uint32_t lane = threadIdx.x & 63, row = lane & 31;
#pragma unroll
    for (int b = 0; b < TR; ++b)
        if (b == j)
#pragma unroll
            for (int i = 0; i < TC; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    part[row * kChunks + ((8 * i + 2 * q + (lane >> 5)) ^ (row & kMask))] =
                        make_float4(acc[i][b][4 * q], acc[i][b][4 * q + 1], acc[i][b][4 * q + 2], acc[i][b][4 * q + 3]);
}

// Epilogues that treat every element by itself derive from this and give
//   ld                      the matrix's columns, and the step from row to row;
//   bias(c)                 what is added to column c (0: nothing);
//   in_words()              whether rows start on 4-byte boundaries;
//   before<N>(elements)     what the elements' put reads of memory, loaded ahead of it;
//   put(elements, bias, z, before)
//                           takes z[x] for element x, its bias in bias[x].
// A wave passes its part of the tile through LDS, 32 rows at a time: there a
// lane wrote four columns of its row at once, here it takes eight of one of
// four rows, so that rows are read and written in whole lines and the columns a
// lane sees stay the same. (Straight from the registers, a lane having four
// columns of each of 32 rows, the code is unrolled for every four, and a
// dropout, bias and activation took 700 us of 8192x4096x16384's 1660.) Chunks of
// four columns are permuted by chunk ^ row.
template <class Self>
struct TileEpilogue {
    static constexpr bool kElementwise = true;  // the K of a product may be cut, and the pieces joined
    __device__ __forceinline__ void one(uint32_t r, uint32_t c, float z) const {
        const Self &self = *static_cast<const Self *>(this);
        const float bias[1] = {self.bias(c)};
        float v[1] = {z};
        const RowRun e{(uint64_t)r * self.ld + c, 1};
        self.put(e, bias, v, self.template before<1>(e));
    }
    // The fp32 kernel's: rows of a 32x32 block, and some of a row.
    __device__ __forceinline__ void block(uint32_t r, uint32_t rows, uint32_t c, float (&z)[16]) const {
        if (r >= rows) return;
        const Self &self = *static_cast<const Self *>(this);
        const float b = self.bias(c);
        const float bias[16] = {b, b, b, b, b, b, b, b, b, b, b, b, b, b, b, b};
        const BlockColumn e{(uint64_t)r * self.ld + c, self.ld, rows - r};
        self.put(e, bias, z, self.template before<16>(e));
    }
    template <int N>
    __device__ __forceinline__ void row(uint32_t r, uint32_t c, uint32_t cols, float (&z)[N]) const {
        const Self &self = *static_cast<const Self *>(this);
        float bias[N];
#pragma unroll
        for (int x = 0; x < N; ++x) bias[x] = self.bias(min(c + x, cols - 1));
        const RowRun e{(uint64_t)r * self.ld + c, min(cols - c, (uint32_t)N)};
        self.put(e, bias, z, self.template before<N>(e));
    }
    // Few rows (product_skinny.hpp): one element, if it is there.
    template <int COLS>
    __device__ __forceinline__ void skinny(uint32_t r, uint32_t c, float z, uint32_t rows, uint32_t cols, uint32_t) const {
        if (r >= rows || c >= cols) return;
        one(r, c, z);
    }
    template <int TR, int TC, int WR, int WC>
    __device__ __forceinline__ void tile(const f32x16 (&acc)[TC][TR], uint32_t r0, uint32_t c0, uint32_t wr0, uint32_t wc0,
                                         uint32_t rows, uint32_t cols, uint32_t, uint32_t, char *lds) const {
        constexpr uint32_t kCols = TC * 32, kLanes = kCols / 8, kStep = kWave / kLanes, kMask = kCols / 4 - 1;
        const Self &self = *static_cast<const Self *>(this);
        const uint32_t lane = threadIdx.x & 63;
        float4 *part = reinterpret_cast<float4 *>(lds) + (threadIdx.x >> 6) * (32 * kCols / 4);
        const uint32_t c = c0 + wc0 + lane % kLanes * 8;
        const bool words = self.in_words();
        float bias[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) bias[i] = self.bias(min(c + i, cols - 1));
        // One copy of the code for all blocks of rows; only the writes to LDS name registers.
#pragma unroll 1
        for (int j = 0; j < TR; ++j) {
            const uint32_t top = r0 + wr0 + 32 * j;
            // A few rows of eights at a time (kStep rows apart), what they read of memory first; the first ones' before the
            // passage through LDS.
            constexpr uint32_t kRows = TC * TR > 4 ? 2 : 4;  // by the registers that the tile leaves
            using Eight = typename Self::template Before<8>;
            const auto eight = [&](uint32_t x) { return RowRun{(uint64_t)(top + x) * self.ld + c, cols - c < 8u ? cols - c : 8u}; };
            const auto ahead = [&](Eight(&to)[kRows], uint32_t x) __attribute__((always_inline)) {
#pragma unroll
                for (uint32_t g = 0; g < kRows; ++g)
                    if (top + x + g * kStep < rows) to[g] = self.template before<8>(eight(x + g * kStep));
            };
            Eight before[kRows] = {};
            if (words && c < cols) ahead(before, lane / kLanes);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            block_to_lds<TR, TC>(acc, j, part);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (words) {
                if (c >= cols) continue;
#pragma unroll 1
                for (uint32_t x = lane / kLanes; x < 32; x += kRows * kStep) {
                    if (x >= kRows * kStep) ahead(before, x);
#pragma unroll
                    for (uint32_t g = 0; g < kRows; ++g) {
                        const uint32_t y = x + g * kStep, at = y * (kCols / 4), chunk = lane % kLanes * 2;
                        if (y >= 32 || top + y >= rows) break;
                        const float4 a = part[at + (chunk ^ (y & kMask))], b = part[at + ((chunk + 1) ^ (y & kMask))];
                        float z[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
                        self.put(eight(y), bias, z, before[g]);
                    }
                }
                continue;
            }
            // Rows that start inside a word: a lane a column, sixteen rows at a time.
#pragma unroll 1
            for (uint32_t col = lane; col < kCols; col += kWave) {
                const uint32_t at = c0 + wc0 + col;
                if (at >= cols) break;
                const float b = self.bias(at);
                const float same[16] = {b, b, b, b, b, b, b, b, b, b, b, b, b, b, b, b};
                const auto sixteen = [&](uint32_t x) {
                    return ColumnRun{(uint64_t)(top + x) * self.ld + at, self.ld, top + x + 16 <= rows ? 16u : top + x < rows ? rows - top - x : 0u};
                };
                const auto first = self.template before<16>(sixteen(0)), second = self.template before<16>(sixteen(16));
#pragma unroll 1
                for (uint32_t x = 0; x < 32; x += 16) {
                    float z[16];
#pragma unroll
                    for (uint32_t i = 0; i < 16; ++i)
                        z[i] = reinterpret_cast<const float *>(part)[((x + i) * (kCols / 4) + ((col / 4) ^ ((x + i) & kMask))) * 4 + col % 4];
                    self.put(sixteen(x), same, z, x == 0 ? first : second);
                }
            }
        }
    }
};

// A split's sums, to be joined.
struct PartialEpilogue : TileEpilogue<PartialEpilogue> {
    float *out;
    uint32_t ld;  // a multiple of eight
    __device__ __forceinline__ PartialEpilogue(float *out, uint32_t ld) : out(out), ld(ld) {}
    __device__ __forceinline__ float bias(uint32_t) const { return 0.0f; }
    __device__ __forceinline__ bool in_words() const { return true; }
    template <int N>
    struct Before {};
    template <int N, class E>
    __device__ __forceinline__ Before<N> before(const E &) const { return {}; }
    template <class E, int N>
    __device__ __forceinline__ void put(const E &e, const float (&)[N], float (&z)[N], const Before<N> &) const {
        if constexpr (N == 8) store8(out, e.first, z);  // also past the last column: ld is whole eights
    }
};

// Tile: its rows and columns, the waves that share them, the slab's depth and how many slabs LDS holds.
template <int BR_, int BC_, int WR_, int WC_, int BK_, int STAGES_>
struct Tile {
    static constexpr int BR = BR_, BC = BC_, WR = WR_, WC = WC_, BK = BK_, STAGES = STAGES_, kThreads = 64 * WR * WC;
};

// LDS of a kernel of these tiles: the slabs, in whose place the epilogue's blocks of 32 rows come after the product.
template <class T, bool ALIGNED>
constexpr uint32_t lds_bytes() {
    constexpr uint32_t slabs = (ALIGNED ? T::STAGES : 2) * (T::BR + T::BC) * T::BK * 2, blocks = T::WR * 32 * T::BC * 4;
    return slabs > blocks ? slabs : blocks;
}

// Workgroup `block` of a product's.
template <class T, bool VMC, bool UMC, bool ALIGNED, class Epi>
__device__ __forceinline__ void product_tile(const ProductArgs &g, const Epi &epi, uint32_t block, char *lds) {
    constexpr int BR = T::BR, BC = T::BC, WR = T::WR, WC = T::WC, BK = T::BK, kThreads = T::kThreads;
    constexpr int kTR = BR / WR / 32, kTC = BC / WC / 32, kSteps = BK / 16, kStages = ALIGNED ? T::STAGES : 2;
    constexpr uint32_t kV = BR * BK * 2, kStage = kV + BC * BK * 2;
    const uint32_t wave = threadIdx.x >> 6;
    const uint32_t tiles = g.tiles_r * g.tiles_c;
    const uint32_t w = xcd_run(block, tiles * g.splits), split = w / tiles;
    uint32_t tr, tc;
    tile_of(w - split * tiles, g.tiles_r, g.tiles_c, tr, tc);
    const uint32_t r0 = tr * BR, c0 = tc * BC, wr0 = wave / WC * (BR / WR), wc0 = wave % WC * (BC / WC);
    const uint32_t kbeg = split * g.k_chunk, kend = min(kbeg + g.k_chunk, g.k);

    f32x16 acc[kTC][kTR];
#pragma unroll
    for (int i = 0; i < kTC; ++i)
#pragma unroll
        for (int j = 0; j < kTR; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

    struct Fragments {
        bf16x8 u[kTC], v[kTR];
    };
    auto read_one = [&](Fragments &f, uint32_t stage, int s, int o) __attribute__((always_inline)) {
        const char *at = lds + stage * kStage;
        if (o < kTC) f.u[o] = fragment<BC, BK, UMC>(at + kV, wc0 + 32 * o, s);
        else f.v[o - kTC] = fragment<BR, BK, VMC>(at, wr0 + 32 * (o - kTC), s);
    };
    auto read = [&](Fragments &f, uint32_t stage, int s) __attribute__((always_inline)) {
#pragma unroll
        for (int o = 0; o < kTC + kTR; ++o) read_one(f, stage, s, o);
    };
    auto multiply = [&](const Fragments &f) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kTC; ++i)
#pragma unroll
            for (int j = 0; j < kTR; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.u[i], f.v[j], acc[i][j], 0, 0, 0);
    };

    if constexpr (ALIGNED) {
        // LDS holds kStages slabs. A wave reads a step's operands while it
        // multiplies the step before; when it has read a slab's last ones and
        // its loads of the next slab have landed, it meets the others, and
        // loads the slab kStages on into the place of the one just read, a few
        // loads a step between the multiplications: issued all at once they
        // hold up every wave of the workgroup for the time that the loads'
        // 64 KB take (4096^3, 256x256 tiles: 115.5 us at once, 108.2 spread).
        if (kbeg < kend) {
            Direct<BR, BK, VMC, kThreads> dv;
            Direct<BC, BK, UMC, kThreads> du;
            constexpr int kLoads = dv.kLoads + du.kLoads;
            dv.init(g.ldv, r0, g.rows);
            if constexpr (kPaired<Epi>) du.init_pairs(g.ldu, c0, epi.half);
            else du.init(g.ldu, c0, g.cols);
            const __bf16 *pv = g.v + (VMC ? (uint64_t)kbeg * g.ldv + r0 : (uint64_t)r0 * g.ldv + kbeg);
            const uint32_t u0 = kPaired<Epi> ? c0 / 2 : c0;
            const __bf16 *pu = g.u + (UMC ? (uint64_t)kbeg * g.ldu + u0 : (uint64_t)u0 * g.ldu + kbeg);
            const uint64_t sv = VMC ? (uint64_t)BK * g.ldv : BK, su = UMC ? (uint64_t)BK * g.ldu : BK;
            const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
            uint32_t left = kend - kbeg, to = base;  // of the slab that is being loaded
            auto load = [&](int i) __attribute__((always_inline)) {
                if (i < dv.kLoads) dv.load(i, pv, left, to);
                else du.load(i - dv.kLoads, pu, left, to + kV);
            };
            auto next_slab = [&]() __attribute__((always_inline)) {
                pv += sv;
                pu += su;
                left = left > (uint32_t)BK ? left - BK : 0;
            };
            // One step: multiplies, and between the multiplications reads the next operands and issues loads from .. end - 1 of
            // the slab. (The compiler would read an operand where it is used, and wait for it.)
            auto step = [&](Fragments &next, uint32_t stage, int s, const Fragments &now, int from, int end) __attribute__((always_inline)) {
                constexpr int kEach = kTC * kTR;
#pragma unroll
                for (int i = 0; i < kTC; ++i)
#pragma unroll
                    for (int j = 0; j < kTR; ++j) {
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(now.u[i], now.v[j], acc[i][j], 0, 0, 0);
                        const int m = i * kTR + j, n = end - from;
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int o = 0; o < kTC + kTR; ++o)
                            if (o * kEach / (kTC + kTR) == m) read_one(next, stage, s, o);
#pragma unroll
                        for (int x = 0; x < n; ++x)
                            if (x * kEach / n == m) load(from + x);
                        __builtin_amdgcn_sched_barrier(0);
                    }
            };
            // Past the end of K the loads write zeros, and go on: their count is what the waits go by.
            static_assert(kSteps % 2 == 0, "steps alternate between two sets of operands");
            constexpr int kParts = kSteps - 1, kPart = (kLoads + kParts - 1) / kParts;  // none in the step before a wait
            constexpr auto part = [](int p) { return p * kPart < kLoads ? p * kPart : kLoads; };
            Fragments f[2];
#pragma unroll
            for (int s = 0; s < kStages; ++s) {
                to = base + s * kStage;
#pragma unroll
                for (int i = 0; i < kLoads; ++i) load(i);
                next_slab();
            }
            await_loads<(kStages - 1) * kLoads>();
            read(f[0], 0, 0);
#pragma unroll
            for (int s = 0; s + 1 < kSteps; ++s) step(f[(s + 1) & 1], 0, s + 1, f[s & 1], 0, 0);
            uint32_t stage = 0;
#pragma unroll 1
            for (uint32_t slabs = (kend - kbeg + BK - 1) / BK; slabs > 1; --slabs) {
                await_loads<(kStages - 2) * kLoads>();
                to = base + stage * kStage;
                stage = stage + 1 == (uint32_t)kStages ? 0 : stage + 1;
                step(f[0], stage, 0, f[1], part(0), part(1));
#pragma unroll
                for (int s = 0; s + 1 < kSteps; ++s) step(f[(s + 1) & 1], stage, s + 1, f[s & 1], part(s + 1), part(s + 2));
                next_slab();
            }
            multiply(f[1]);
            await_loads<0>();  // LDS is the epilogue's now
        }
    } else {
        // Two slabs of LDS and two in registers: a slab's loads are issued two
        // slabs ahead and stored to LDS one ahead.
        if (kbeg < kend) {
            struct Slab {
                Staged<BR, BK, VMC, kThreads> v;
                Staged<BC, BK, UMC, kThreads> u;
            };
            auto load = [&](Slab &s, uint32_t k0) __attribute__((always_inline)) {
                if (k0 >= kend) return;
                s.v.load(g.v, g.ldv, r0, g.rows, k0, kend);
                if constexpr (kPaired<Epi>) s.u.load_pairs(g.u, g.ldu, c0, epi.half, k0, kend);
                else s.u.load(g.u, g.ldu, c0, g.cols, k0, kend);
            };
            auto store = [&](const Slab &s, uint32_t stage) __attribute__((always_inline)) {
                s.v.store(lds + stage * kStage);
                s.u.store(lds + stage * kStage + kV);
            };
            Slab a, b;
            load(a, kbeg);
            load(b, kbeg + BK);
            store(a, 0);
            __syncthreads();
            // Slab k0 is in LDS and the next one in `next`; the one after goes to `after`.
            auto slab = [&](uint32_t k0, uint32_t stage, Slab &after, const Slab &next) __attribute__((always_inline)) {
                load(after, k0 + 2 * BK);
                __builtin_amdgcn_sched_barrier(0);
                Fragments f;
#pragma unroll
                for (int s = 0; s < kSteps; ++s) {
                    read(f, stage, s);
                    multiply(f);
                }
                __builtin_amdgcn_sched_barrier(0);
                if (k0 + BK < kend) store(next, stage ^ 1);
                __syncthreads();
            };
#pragma unroll 1
            for (uint32_t k0 = kbeg; k0 < kend; k0 += 2 * BK) {
                slab(k0, 0, a, b);
                if (k0 + BK < kend) slab(k0 + BK, 1, b, a);
            }
        }
    }

    if (g.splits > 1) {
        const PartialEpilogue part{g.partial + (uint64_t)split * g.rows * g.ldp, g.ldp};
        part.template tile<kTR, kTC, WR, WC>(acc, r0, c0, wr0, wc0, g.rows, g.cols, tr, tc, lds);
        return;
    }
    epi.template tile<kTR, kTC, WR, WC>(acc, r0, c0, wr0, wc0, g.rows, g.cols, tr, tc, lds);
}

template <class T, bool VMC, bool UMC, bool ALIGNED, class Epi>
__global__ __launch_bounds__(T::kThreads, 2) void product_kernel(ProductArgs g, Epi epi) {
    __shared__ __align__(1024) char lds[lds_bytes<T, ALIGNED>()];
    product_tile<T, VMC, UMC, ALIGNED>(g, epi, g.first_block + blockIdx.x, lds);
}

// A backward pass's two products in one launch: a's tiles (u row-contiguous
// alone) and b's (both operands), a's in the first workgroups or in the last.
template <class T, class Epi>
__global__ __launch_bounds__(T::kThreads, 2) void product_pair_kernel(ProductArgs a, Epi epi_a, ProductArgs b, Epi epi_b, uint32_t tiles_a,
                                                                     bool a_first) {
    __shared__ __align__(1024) char lds[lds_bytes<T, true>()];
    const uint32_t first = a_first ? tiles_a : gridDim.x - tiles_a, block = blockIdx.x < first ? blockIdx.x : blockIdx.x - first;
    if ((blockIdx.x < first) == a_first) product_tile<T, false, true, true>(a, epi_a, block, lds);
    else product_tile<T, true, true, true>(b, epi_b, block, lds);
}

// The join of a split product: adds eight columns' partials in f64 and passes
// them to the epilogue. GROUPS threads share them, each taking every GROUPSth
// split, and are added in order: one thread up to four splits, eight beyond
// (5x368 of 24 splits 9.7 us with one).
template <int GROUPS, class Epi>
__global__ __launch_bounds__(kBlock) void join_kernel(ProductArgs g, Epi epi) {
    constexpr uint32_t kItems = kBlock / GROUPS;
    const uint32_t eights = g.ldp / 8, group = threadIdx.x / kItems, e = blockIdx.x * kItems + threadIdx.x % kItems;
    const bool in = e < g.rows * eights;
    const uint32_t r = e / eights, c = (e - r * eights) * 8;
    double s[8] = {};
    if (in) {
        const float *from = g.partial + (uint64_t)r * g.ldp + c;
#pragma unroll 4
        for (uint32_t p = group; p < g.splits; p += GROUPS) {
            const float4 *at = reinterpret_cast<const float4 *>(from + (uint64_t)p * g.rows * g.ldp);
            const float4 x = at[0], y = at[1];
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] += (double)lane(i < 4 ? x : y, i & 3);
        }
    }
    if constexpr (GROUPS > 1) {
        __shared__ double sums[GROUPS][8][kItems];
#pragma unroll
        for (int i = 0; i < 8; ++i) sums[group][i][threadIdx.x % kItems] = s[i];
        __syncthreads();
        if (group != 0) return;
#pragma unroll
        for (int p = 1; p < GROUPS; ++p)
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] += sums[p][i][threadIdx.x];
    }
    if (!in) return;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)s[i];
    epi.row(r, c, g.cols, v);
}

}  // namespace
}  // namespace dkz
