// product.hpp -- bf16 matrix products with an epilogue, fp32 sums:
//     out(r, c) = epilogue(sum over k of v(r, k) * u(c, k)).
//
// An operand is k-contiguous (element (row, k) at p[row * ld + k]) or
// row-contiguous (at p[k * ld + row]). v_mfma_f32_32x32x16_bf16 takes u as its
// A operand, so that a lane holds four consecutive columns c of one row r in
// consecutive registers: the epilogues store four at a time.
//
// A workgroup owns BR rows x BC columns, its waves WR x WC parts of that. K
// advances in slabs of 64: while the waves multiply one slab out of LDS, the
// next is on its way. In LDS a k-contiguous operand's slab is [row][64 k], its
// 16-byte chunks permuted by chunk ^ (row & 7), so that the eight rows that are
// read together lie in different banks; a lane's operand (eight k of its row) is
// one 128-bit read. A row-contiguous one is [k][rows], its chunks permuted by
// chunk ^ 4 * (k & 3), and read transposed (ds_read_b64_tr_b16: sixteen lanes
// take a block of four k and sixteen rows, each lane the four k of one row).
#pragma once

#include "dense_internal.hpp"

namespace dkz {
namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef short s16x8u __attribute__((ext_vector_type(8), aligned(2)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr uint32_t kSlabK = 64;

struct ProductArgs {
    const __bf16 *v, *u;  // row side, column side
    uint32_t ldv, ldu;
    uint32_t rows, cols, k;
    uint32_t tiles_r, tiles_c, splits, k_chunk;  // k_chunk: a split's K, a multiple of kSlabK
    float *partial;                              // splits > 1: [splits][rows][ldp]
    uint32_t ldp;
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

// A slab of R rows of an operand on its way to LDS through registers, whatever
// its alignment. MC: row-contiguous.
template <int R, bool MC, int THREADS>
struct Staged {
    static constexpr int kChunks = R * (int)kSlabK / 8 / THREADS;
    static_assert(kChunks * 8 * THREADS == R * (int)kSlabK, "whole chunks a thread");
    s16x8 v[kChunks];

    // Rows past `rows` and k past `kend` read as 0.
    __device__ __forceinline__ void load(const __bf16 *p, uint32_t ld, uint32_t r0, uint32_t rows, uint32_t k0, uint32_t kend) {
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const uint32_t c = threadIdx.x + i * THREADS;
            const uint32_t row = r0 + (MC ? c % (R / 8) * 8 : c / 8), k = k0 + (MC ? c / (R / 8) : c % 8 * 8);
            const short *at = reinterpret_cast<const short *>(p) + (MC ? (uint64_t)k * ld + row : (uint64_t)row * ld + k);
            s16x8 x = {};
            if (row < rows && k < kend) {
                const uint32_t n = MC ? rows - row : kend - k;
                if (n >= 8) {
                    x = *reinterpret_cast<const s16x8u *>(at);
                } else {
#pragma unroll
                    for (int j = 0; j < 7; ++j)
                        if (j < (int)n) x[j] = at[j];
                }
            }
            v[i] = x;
        }
    }
    __device__ __forceinline__ void store(char *lds) const {
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const uint32_t c = threadIdx.x + i * THREADS;
            const uint32_t line = MC ? c / (R / 8) : c / 8, chunk = MC ? c % (R / 8) : c % 8;
            const uint32_t to = MC ? line * (R / 8) + (chunk ^ ((line & 3) * 4 & (R / 8 - 1))) : line * 8 + (chunk ^ (line & 7));
            *reinterpret_cast<s16x8 *>(lds + to * 16) = v[i];
        }
    }
};

// Rows row .. row + 31 of a slab in LDS, k 16 * step + 8 * (lane / 32) + 0 .. 7, as an MFMA operand.
template <int R, bool MC>
__device__ __forceinline__ bf16x8 fragment(const char *lds, uint32_t row, int step) {
    const uint32_t lane = threadIdx.x & 63;
    if constexpr (!MC) {
        const uint32_t r = row + (lane & 31), chunk = 2 * step + (lane >> 5);
        return *reinterpret_cast<const bf16x8 *>(lds + r * 128 + ((chunk ^ (r & 7)) * 16));
    } else {
        // Lane a of a group of sixteen names four rows of k line a / 4.
        const uint32_t a = lane & 15, k = 16 * step + 8 * (lane >> 5) + a / 4, r = row + (lane & 16) + 4 * (a & 3);
        const uint32_t at = k * (R * 2) + (((r >> 3) ^ ((k & 3) * 4 & (R / 8 - 1))) * 16) + (r & 4) * 2;
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(lds + at));
        const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(lds + at + 4 * R * 2));
        const s16x8 both = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
        return __builtin_bit_cast(bf16x8, both);
    }
}

// acc[i][j][e] is (r, c) = (32 * j + lane % 32, 32 * i + 8 * (e / 4) + 4 * (lane / 32) + e % 4) of the wave's part.
template <int BR, int BC, int WR, int WC, bool VMC, bool UMC, class Epi>
__global__ __launch_bounds__(64 * WR * WC) void product_kernel(ProductArgs g, Epi epi) {
    constexpr int kThreads = 64 * WR * WC, kTR = BR / WR / 32, kTC = BC / WC / 32;
    constexpr int kV = BR * kSlabK * 2, kU = BC * kSlabK * 2;
    __shared__ __align__(16) char lds[2 * (kV + kU)];
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const uint32_t tiles = g.tiles_r * g.tiles_c;
    const uint32_t w = xcd_run(blockIdx.x, tiles * g.splits), split = w / tiles;
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

    Staged<BR, VMC, kThreads> sv;
    Staged<BC, UMC, kThreads> su;
    if (kbeg < kend) {
        sv.load(g.v, g.ldv, r0, g.rows, kbeg, kend);
        su.load(g.u, g.ldu, c0, g.cols, kbeg, kend);
        sv.store(lds);
        su.store(lds + kV);
        __syncthreads();
        uint32_t cur = 0;
#pragma unroll 1
        for (uint32_t k0 = kbeg; k0 < kend; k0 += kSlabK, cur ^= 1) {
            const bool more = k0 + kSlabK < kend;
            if (more) {
                sv.load(g.v, g.ldv, r0, g.rows, k0 + kSlabK, kend);
                su.load(g.u, g.ldu, c0, g.cols, k0 + kSlabK, kend);
            }
            const char *lv = lds + cur * (kV + kU), *lu = lv + kV;
#pragma unroll
            for (int s = 0; s < (int)kSlabK / 16; ++s) {
                bf16x8 fu[kTC], fv[kTR];
#pragma unroll
                for (int i = 0; i < kTC; ++i) fu[i] = fragment<BC, UMC>(lu, wc0 + 32 * i, s);
#pragma unroll
                for (int j = 0; j < kTR; ++j) fv[j] = fragment<BR, VMC>(lv, wr0 + 32 * j, s);
#pragma unroll
                for (int i = 0; i < kTC; ++i)
#pragma unroll
                    for (int j = 0; j < kTR; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fu[i], fv[j], acc[i][j], 0, 0, 0);
            }
            if (more) {
                char *to = lds + (cur ^ 1) * (kV + kU);
                sv.store(to);
                su.store(to + kV);
            }
            __syncthreads();
        }
    }

    if (g.splits > 1) {
        float *to = g.partial + (uint64_t)split * g.rows * g.ldp;
#pragma unroll
        for (int j = 0; j < kTR; ++j) {
            const uint32_t r = r0 + wr0 + 32 * j + (lane & 31);
            if (r >= g.rows) continue;
#pragma unroll
            for (int i = 0; i < kTC; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint32_t c = c0 + wc0 + 32 * i + 8 * q + 4 * (lane >> 5);
                    if (c < g.cols)
                        *reinterpret_cast<float4 *>(to + (uint64_t)r * g.ldp + c) =
                            make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
                }
        }
        return;
    }
    epi.template tile<kTR, kTC, WR, WC>(acc, r0, c0, wr0, wc0, g.rows, g.cols, tr, tc, lds);
}

// The join of a split product: adds a quad's partials in split order, in f64, and passes it to the epilogue.
template <class Epi>
__global__ __launch_bounds__(kBlock) void join_kernel(ProductArgs g, Epi epi) {
    const uint32_t quads = g.ldp / 4, q = blockIdx.x * kBlock + threadIdx.x;
    if (q >= g.rows * quads) return;
    const uint32_t r = q / quads, c = (q - r * quads) * 4;
    const float *from = g.partial + (uint64_t)r * g.ldp + c;
    double s[4] = {};
    for (uint32_t p = 0; p < g.splits; ++p) {
        const float4 x = *reinterpret_cast<const float4 *>(from + (uint64_t)p * g.rows * g.ldp);
        s[0] += (double)x.x;
        s[1] += (double)x.y;
        s[2] += (double)x.z;
        s[3] += (double)x.w;
    }
    epi.quad(r, c, g.cols, make_float4((float)s[0], (float)s[1], (float)s[2], (float)s[3]));
}

// Epilogues that treat every element by itself derive from this: quad(r, c,
// cols, v) takes columns c .. c + 3 of row r, of which those below cols exist.
template <class Self>
struct QuadEpilogue {
    template <int TR, int TC, int WR, int WC>
    __device__ __forceinline__ void tile(const f32x16 (&acc)[TC][TR], uint32_t r0, uint32_t c0, uint32_t wr0, uint32_t wc0,
                                         uint32_t rows, uint32_t cols, uint32_t, uint32_t, char *) const {
        const uint32_t lane = threadIdx.x & 63;
#pragma unroll
        for (int j = 0; j < TR; ++j) {
            const uint32_t r = r0 + wr0 + 32 * j + (lane & 31);
            if (r >= rows) continue;
#pragma unroll
            for (int i = 0; i < TC; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint32_t c = c0 + wc0 + 32 * i + 8 * q + 4 * (lane >> 5);
                    if (c < cols)
                        static_cast<const Self *>(this)->quad(
                            r, c, cols, make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]));
                }
        }
    }
};

// How a product is cut: tiles of br x bc, K in `splits` ranges of k_chunk.
struct ProductPlan {
    uint32_t br, bc, splits, k_chunk;
    uint64_t partial_bytes(uint64_t rows, uint64_t cols) const {
        return splits > 1 ? padded(4 * (uint64_t)splits * rows * round_up(cols, 4)) : 0;
    }
};

inline ProductPlan plan_product(uint64_t rows, uint64_t cols, uint64_t k, bool may_split) {
    (void)rows;
    (void)cols;
    (void)may_split;
    return {128, 128, 1, (uint32_t)round_up(k, kSlabK)};
}

template <bool VMC, bool UMC, class Epi>
int run_product(const char *name, const __bf16 *v, uint64_t ldv, const __bf16 *u, uint64_t ldu, uint64_t rows, uint64_t cols,
                uint64_t k, const ProductPlan &p, float *partial, const Epi &epi) {
    if (rows == 0 || cols == 0) return 0;
    ProductArgs g{v, u, (uint32_t)ldv, (uint32_t)ldu, (uint32_t)rows, (uint32_t)cols, (uint32_t)k, div_up(rows, p.br),
                  div_up(cols, p.bc), p.splits, p.k_chunk, partial, (uint32_t)round_up(cols, 4)};
    const dim3 grid((uint32_t)((uint64_t)g.tiles_r * g.tiles_c * g.splits));
    DKZ_TRY(launch(name, product_kernel<128, 128, 2, 2, VMC, UMC, Epi>, grid, dim3(256), g, epi));
    return 0;
}

}  // namespace
}  // namespace dkz
