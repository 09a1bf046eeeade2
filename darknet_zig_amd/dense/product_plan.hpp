// product_plan.hpp -- which kernel, tiles and K ranges a bf16 product takes, and its launches.
#pragma once

#include <algorithm>

#include "dense_internal.hpp"
#include "product.hpp"
#include "product_skinny.hpp"

namespace dkz {
namespace {

typedef Tile<256, 256, 4, 2, 64, 2> Tile256;
typedef Tile<128, 128, 2, 2, 64, 4> Tile128;
typedef Tile<64, 128, 2, 2, 64, 3> Tile64x128;
typedef Tile<64, 64, 2, 2, 64, 3> Tile64;

// The kinds of tile and what a slab of 64 k costs a compute unit that has
// 1, 2 .. `occupancy` of them (what LDS has room for), in us with all compute
// units at work: measured over K 4096 at 4096^2 (256x256: 108 us), 1024x4096
// (128x128: 36.5; two slabs in LDS and two a compute unit are 4 us slower),
// 512x4096 and 1024x4096 (64x128: 24.5 and 41.6), 256x4096 .. 1024x4096 (64x64:
// 19.0, 26.7, 51.6).
struct TileKind {
    uint32_t br, bc, wr, wc, occupancy;
    float slab[3], fixed;
};
constexpr TileKind kTileKinds[] = {{256, 256, 4, 2, 1, {1.62f}, 6.0f},
                                   {128, 128, 2, 2, 1, {0.52f}, 4.0f},
                                   {64, 128, 2, 2, 2, {0.32f, 0.59f}, 4.0f},
                                   {64, 64, 2, 2, 3, {0.24f, 0.37f, 0.55f}, 4.0f}};
constexpr uint32_t kComputeUnits = 256;

// How a product is cut: tiles of br x bc, each by wr x wc waves; K in `splits`
// ranges of k_chunk. br 0: the kernel for few rows.
struct ProductPlan {
    uint32_t br, bc, wr, wc, splits, k_chunk;
    bool skinny() const { return br == 0; }
    uint64_t partial_bytes(uint64_t rows, uint64_t cols) const {
        return splits > 1 ? padded(4 * (uint64_t)splits * rows * round_up(cols, 8)) : 0;
    }
    // How many parts of a row, and of a column, an epilogue sees one at a time.
    uint64_t row_parts(uint64_t cols) const { return skinny() ? div_up(cols, skinny_columns(cols)) : (uint64_t)div_up(cols, bc) * wc; }
    uint64_t column_parts(uint64_t rows) const { return skinny() ? rows : (uint64_t)div_up(rows, br) * wr; }
};

// nt: both operands with k contiguous. The least time over the kinds of tile and
// the ways to cut K, each range at least four slabs long: rounds of the chip x
// slabs x a slab's time; ranges add their partials' way out and back and the
// launch that joins them.
inline ProductPlan plan_product(uint64_t rows, uint64_t cols, uint64_t k, bool nt, bool may_split) {
    if (nt && rows <= kSkinnyRows) return {0, 0, 0, 0, 1, 0};
    const uint64_t slabs = (k + 63) / 64;
    constexpr uint32_t kSplits[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32, 48, 64};
    ProductPlan best{};
    float least = 1e30f;
    for (const TileKind &t : kTileKinds) {
        const uint64_t tiles = (uint64_t)div_up(rows, t.br) * div_up(cols, t.bc), slots = (uint64_t)kComputeUnits * t.occupancy;
        for (const uint32_t want : kSplits) {
            const uint64_t chunk = std::max<uint64_t>((slabs + want - 1) / want, 1), splits = std::max<uint64_t>((slabs + chunk - 1) / chunk, 1);
            const uint64_t groups = tiles * splits;
            if (want > 1 && (!may_split || chunk < 4 || groups > 4 * kComputeUnits)) break;
            const uint64_t rounds = groups / slots, rest = groups % slots;
            float us = (float)rounds * ((float)chunk * t.slab[t.occupancy - 1] + t.fixed);
            if (rest) us += (float)chunk * t.slab[(rest - 1) / kComputeUnits] + t.fixed;
            if (splits > 1) us += 3.0f + 8e-6f * (float)(splits * rows * cols) / 4.0f;
            if (us < least) {
                least = us;
                best = {t.br, t.bc, t.wr, t.wc, (uint32_t)splits, (uint32_t)(chunk * 64)};
            }
        }
    }
    return best;
}

// Whether an operand's rows start on 16-byte boundaries and are within the
// loads' 32-bit offsets of each other. A k-contiguous one is whole chunks long
// (`k` of them, or zeros to the end of the last).
template <bool MC>
inline bool direct_ok(const void *p, uint64_t ld, uint64_t k, bool zeros) {
    return aligned16(p) && ld % 8 == 0 && ld < (1u << 22) && (MC || k % 8 == 0 || zeros);
}

template <class T, bool VMC, bool UMC, class Epi>
int launch_product(const char *name, dim3 grid, bool aligned, const ProductArgs &g, const Epi &epi) {
    const dim3 block(T::kThreads);
    if (aligned) return launch(name, product_kernel<T, VMC, UMC, true, Epi>, grid, block, g, epi);
    return launch(name, product_kernel<T, VMC, UMC, false, Epi>, grid, block, g, epi);
}

// zeros: rows of v end in zeros up to a whole chunk. `partial` has the plan's partial_bytes.
template <bool VMC, bool UMC, class Epi>
int run_product(const char *name, const __bf16 *v, uint64_t ldv, const __bf16 *u, uint64_t ldu, uint64_t rows, uint64_t cols,
                uint64_t k, const ProductPlan &p, float *partial, const Epi &epi, bool zeros = false) {
    if (rows == 0 || cols == 0) return 0;
    if constexpr (!VMC && !UMC)
        if (p.skinny()) return run_skinny(name, v, ldv, u, ldu, rows, cols, k, epi);
    ProductArgs g{v, u, (uint32_t)ldv, (uint32_t)ldu, (uint32_t)rows, (uint32_t)cols, (uint32_t)k, div_up(rows, p.br),
                  div_up(cols, p.bc), p.splits, p.k_chunk, partial, (uint32_t)round_up(cols, 8)};
    const uint64_t groups = (uint64_t)g.tiles_r * g.tiles_c * g.splits;
    DKZ_REQUIRE(groups <= 0x7fffffffull);
    const dim3 grid((uint32_t)groups);
    const bool aligned = direct_ok<VMC>(v, ldv, k, zeros) && direct_ok<UMC>(u, ldu, k, false);
    if (p.br == 256) DKZ_TRY((launch_product<Tile256, VMC, UMC>(name, grid, aligned, g, epi)));
    else if (p.br == 128) DKZ_TRY((launch_product<Tile128, VMC, UMC>(name, grid, aligned, g, epi)));
    else if (p.bc == 128) DKZ_TRY((launch_product<Tile64x128, VMC, UMC>(name, grid, aligned, g, epi)));
    else DKZ_TRY((launch_product<Tile64, VMC, UMC>(name, grid, aligned, g, epi)));
    if constexpr (Epi::kElementwise)
        if (g.splits > 1)
            return launch(name, join_kernel<Epi>, dim3(div_up((uint64_t)g.rows * (g.ldp / 8), kBlock)), dim3(kBlock), g, epi);
    return 0;
}

}  // namespace
}  // namespace dkz
