// product_plan.hpp -- which kernel, tiles and K ranges a bf16 product takes, and its launches.
#pragma once

#include "dense_internal.hpp"
#include "product.hpp"
#include "product_skinny.hpp"

namespace dkz {
namespace {

typedef Tile<256, 256, 4, 2, 64, 2> Tile256;
typedef Tile<128, 128, 2, 2, 64, 2> Tile128;

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

// nt: both operands with k contiguous.
inline ProductPlan plan_product(uint64_t rows, uint64_t cols, uint64_t k, bool nt, bool may_split) {
    (void)may_split;
    if (nt && rows <= kSkinnyRows) return {0, 0, 0, 0, 1, 0};
    const uint32_t t = rows > 128 && cols > 128 && div_up(rows, 256) * div_up(cols, 256) >= 200 ? 256 : 128;
    return {t, t, t == 256 ? 4u : 2u, 2, 1, (uint32_t)round_up(k, 64)};
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

// zeros: rows of v end in zeros up to a whole chunk.
template <bool VMC, bool UMC, class Epi>
int run_product(const char *name, const __bf16 *v, uint64_t ldv, const __bf16 *u, uint64_t ldu, uint64_t rows, uint64_t cols,
                uint64_t k, const ProductPlan &p, float *partial, const Epi &epi, bool zeros = false) {
    if (rows == 0 || cols == 0) return 0;
    if constexpr (!VMC && !UMC)
        if (p.skinny()) return run_skinny(name, v, ldv, u, ldu, rows, cols, k, epi);
    ProductArgs g{v, u, (uint32_t)ldv, (uint32_t)ldu, (uint32_t)rows, (uint32_t)cols, (uint32_t)k, div_up(rows, p.br),
                  div_up(cols, p.bc), p.splits, p.k_chunk, partial, (uint32_t)round_up(cols, 8)};
    const dim3 grid((uint32_t)((uint64_t)g.tiles_r * g.tiles_c * g.splits));
    const bool aligned = direct_ok<VMC>(v, ldv, k, zeros) && direct_ok<UMC>(u, ldu, k, false);
    if (p.br == 256) return launch_product<Tile256, VMC, UMC>(name, grid, aligned, g, epi);
    return launch_product<Tile128, VMC, UMC>(name, grid, aligned, g, epi);
}

}  // namespace
}  // namespace dkz
