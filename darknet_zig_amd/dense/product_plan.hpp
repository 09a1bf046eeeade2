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
// 19.0, 26.7, 51.6). `fixed`: a round's first loads and its stores.
struct TileKind {
    uint32_t br, bc, wr, wc, occupancy;
    float slab[3], fixed;
};
constexpr TileKind kTileKinds[] = {{256, 256, 4, 2, 1, {1.62f}, 4.0f},
                                   {128, 128, 2, 2, 1, {0.52f}, 1.2f},
                                   {64, 128, 2, 2, 2, {0.32f, 0.59f}, 1.0f},
                                   {64, 64, 2, 2, 3, {0.24f, 0.37f, 0.55f}, 1.0f}};
constexpr float kLaunchUs = 3.0f, kPartialBytesUs = 4e6f;  // a launch, and bytes of partials a us
constexpr uint32_t kComputeUnits = 256;
// What cutting K adds: the partials' way out and back and the launch that joins them.
inline float join_us(uint64_t splits, uint64_t rows, uint64_t cols) {
    return kLaunchUs + 2 * 4.0f / kPartialBytesUs * (float)(splits * rows * cols);
}

// How a product is cut: tiles of br x bc, each by wr x wc waves; K in `splits`
// ranges of k_chunk. br 0: the kernel for few rows, bc its columns a workgroup.
struct ProductPlan {
    uint32_t br, bc, wr, wc, splits, k_chunk;
    bool direct;  // operands straight to LDS
    float us;     // its time, without a launch
    bool skinny() const { return br == 0; }
    uint64_t partial_bytes(uint64_t rows, uint64_t cols) const {
        return splits > 1 ? padded(4 * (uint64_t)splits * rows * round_up(cols, 8)) : 0;
    }
    // How many parts of a row, and of a column, an epilogue sees one at a time.
    uint64_t row_parts(uint64_t cols) const { return (uint64_t)div_up(cols, bc) * (skinny() ? 1 : wc); }
    uint64_t column_parts(uint64_t rows) const { return skinny() ? rows : (uint64_t)div_up(rows, br) * wr; }
};

// Whether an operand's rows start on 16-byte boundaries and are within the
// loads' 32-bit offsets of each other. (Rows longer than k end in zeros, all of
// them the workspace's.)
inline bool direct_ok(const void *p, uint64_t ld) { return aligned16(p) && ld % 8 == 0 && ld < (1u << 22); }
inline bool operands_direct(const __bf16 *v, uint64_t ldv, const __bf16 *u, uint64_t ldu) { return direct_ok(v, ldv) && direct_ok(u, ldu); }

// nt: both operands with k contiguous; direct: operands_direct. The least time
// over the kinds of tile and the ways to cut K, each range at least four slabs long: rounds of the chip x
// slabs x a slab's time; ranges add their partials' way out and back and the
// launch that joins them.
inline ProductPlan plan_product(uint64_t rows, uint64_t cols, uint64_t k, bool nt, bool may_split, bool direct) {
    if (nt && few_rows(rows)) return {0, skinny_columns(rows, cols, k), 0, 0, 1, 0, false, 0.0f};
    const uint64_t slabs = (k + 63) / 64;
    constexpr uint32_t kSplits[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32, 48, 64};
    ProductPlan best{};
    float least = 1e30f;
    for (const TileKind &t : kTileKinds) {
        if (!direct && (t.br != t.bc || t.br == 256)) continue;  // the kernel that goes through registers has two kinds
        const uint64_t tiles = (uint64_t)div_up(rows, t.br) * div_up(cols, t.bc), slots = (uint64_t)kComputeUnits * t.occupancy;
        for (const uint32_t want : kSplits) {
            const uint64_t chunk = std::max<uint64_t>((slabs + want - 1) / want, 1), splits = std::max<uint64_t>((slabs + chunk - 1) / chunk, 1);
            const uint64_t groups = tiles * splits;
            if (want > 1 && (!may_split || chunk < 4 || groups > 4 * kComputeUnits)) break;
            const uint64_t rounds = groups / slots, rest = groups % slots;
            float us = (float)rounds * ((float)chunk * t.slab[t.occupancy - 1] + t.fixed);
            if (rest) us += (float)chunk * t.slab[(rest - 1) / kComputeUnits] + t.fixed;
            if (splits > 1) us += join_us(splits, rows, cols);
            if (us < least) {
                least = us;
                best = {t.br, t.bc, t.wr, t.wc, (uint32_t)splits, (uint32_t)(chunk * 64), direct, us};
            }
        }
    }
    return best;
}

// ---- rows that are no whole chunks ----
//
// Matrices with k contiguous and k % 8 != 0 are copied to the workspace in rows
// of whole chunks that end in zeros, for the products that read them once a
// tile: 777x1001x2503 with its epilogue took 86 us through registers, where loads
// at odd elements and the shifts at rows' ends hold up the products, and 44 us
// by copies (5 us of them). Operands whose rows are whole chunks and whose base
// is off a 16-byte boundary go through registers (4096^3 270 us).

inline uint64_t packed_ld(uint64_t k) { return round_up(k, 8); }
inline uint64_t packed_bytes(uint64_t rows, uint64_t k) { return k % 8 == 0 ? 0 : padded(2 * rows * packed_ld(k)); }

// What is to be copied: rows_a rows of a, then rows_b of b, in chunks.
struct PackArgs {
    const __bf16 *a;
    uint32_t rows_a;
    __bf16 *to_a;
    const __bf16 *b;
    uint32_t rows_b;
    __bf16 *to_b;
    uint32_t k;
    FastDiv chunks;  // of a row
    uint64_t count() const { return ((uint64_t)rows_a + rows_b) * chunks.d; }
};

// Chunk `at` of the copies.
__device__ __forceinline__ void pack_chunk(const PackArgs &g, uint32_t at) {
    const uint32_t end_a = g.rows_a * g.chunks.d;
    if (at >= end_a + g.rows_b * g.chunks.d) return;
    const __bf16 *from = at < end_a ? g.a : g.b;
    __bf16 *to = at < end_a ? g.to_a : g.to_b;
    at -= at < end_a ? 0 : end_a;
    const uint32_t row = fdiv(at, g.chunks), c = (at - row * g.chunks.d) * 8;
    const short *p = reinterpret_cast<const short *>(from) + (uint64_t)row * g.k + c;
    s16x8 v = {};
    if (c + 8 <= g.k) {
        v = load_shifted(p);
    } else {
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (c + i < g.k) v[i] = p[i];
    }
    reinterpret_cast<s16x8 *>(to)[at] = v;
}
// A thread a chunk.
__global__ __launch_bounds__(kBlock) void pack_kernel(PackArgs g) { pack_chunk(g, blockIdx.x * kBlock + threadIdx.x); }

// A matrix as the products take it.
struct Matrix {
    const __bf16 *p;
    uint64_t ld;
};

// a and b (null: left out) become copies in the workspace where their rows are no whole chunks; what is then to be copied.
inline PackArgs pack_args(Matrix &a, uint64_t rows_a, Matrix &b, uint64_t rows_b, uint64_t k, Workspace &ws) {
    if (k % 8 == 0) return {};
    const uint64_t ld = packed_ld(k), na = a.p != nullptr ? rows_a : 0, nb = b.p != nullptr ? rows_b : 0;
    __bf16 *to_a = ws.take<__bf16>(packed_bytes(rows_a, k) / 2), *to_b = ws.take<__bf16>(packed_bytes(rows_b, k) / 2);
    const PackArgs g{a.p, (uint32_t)na, to_a, b.p, (uint32_t)nb, to_b, (uint32_t)k, make_fastdiv((uint32_t)(ld / 8))};
    if (na) a = {to_a, ld};
    if (nb) b = {to_b, ld};
    return g;
}
inline int pack(hipStream_t stream, Matrix &a, uint64_t rows_a, Matrix &b, uint64_t rows_b, uint64_t k, Workspace &ws) {
    const PackArgs g = pack_args(a, rows_a, b, rows_b, k, ws);
    return g.count() != 0 ? launch_on(stream, "pack", pack_kernel, dim3(div_up(g.count(), kBlock)), dim3(kBlock), g) : 0;
}

// A size that a workspace is planned by, whatever the alignment of the operands.
template <class F>
inline uint64_t most_of_plans(uint64_t rows, uint64_t cols, uint64_t k, bool nt, bool may_split, F f) {
    return std::max<uint64_t>(f(plan_product(rows, cols, k, nt, may_split, true)), f(plan_product(rows, cols, k, nt, may_split, false)));
}
inline uint64_t most_partial_bytes(uint64_t rows, uint64_t cols, uint64_t k, bool nt) {
    return most_of_plans(rows, cols, k, nt, true, [&](const ProductPlan &p) { return p.partial_bytes(rows, cols); });
}

// A bf16 product's operands and sizes.
struct Product {
    const __bf16 *v;
    uint64_t ldv;
    const __bf16 *u;
    uint64_t ldu, rows, cols, k;
    bool direct() const { return operands_direct(v, ldv, u, ldu); }
};

inline ProductArgs product_args(const Product &x, const ProductPlan &p, float *partial) {
    return {x.v, x.u, (uint32_t)x.ldv, (uint32_t)x.ldu, (uint32_t)x.rows, (uint32_t)x.cols, (uint32_t)x.k, div_up(x.rows, p.br),
            div_up(x.cols, p.bc), p.splits, p.k_chunk, partial, (uint32_t)round_up(x.cols, 8), 0};
}

// Workgroups of a launch at most: its threads are counted in 32 bits, and 2^38 logits in tiles of 128x128 are 2^24
// workgroups of 256. A product of more takes several launches. (A multiple of the XCDs, so that xcd_run goes on as it was.)
constexpr uint64_t kMostGroups = 1ull << 22;

// Where K was cut.
template <class Epi>
int join_product(hipStream_t stream, const char *name, const ProductArgs &g, const Epi &epi) {
    const uint64_t eights = (uint64_t)g.rows * (g.ldp / 8);
    if (g.splits > 4) return launch_on(stream, name, join_kernel<8, Epi>, dim3(div_up(eights, kBlock / 8)), dim3(kBlock), g, epi);
    if (g.splits > 1) return launch_on(stream, name, join_kernel<1, Epi>, dim3(div_up(eights, kBlock)), dim3(kBlock), g, epi);
    return 0;
}

// `partial` has the plan's partial_bytes.
template <bool VMC, bool UMC, class Epi>
int run_product(hipStream_t stream, const char *name, const Product &x, const ProductPlan &p, float *partial, const Epi &epi) {
    if (x.rows == 0 || x.cols == 0) return 0;
    if constexpr (!VMC && !UMC)
        if (p.skinny()) return run_skinny(stream, name, x.v, x.ldv, x.u, x.ldu, x.rows, x.cols, x.k, p.bc, epi);
    ProductArgs g = product_args(x, p, partial);
    const uint64_t groups = (uint64_t)g.tiles_r * g.tiles_c * g.splits;
    DKZ_REQUIRE(groups <= 0x7fffffffull);
    const dim3 four(256);
    for (uint64_t first = 0; first < groups; first += kMostGroups) {
        g.first_block = (uint32_t)first;
        const dim3 grid((uint32_t)std::min(groups - first, kMostGroups));
        if (!p.direct) {
            if (p.br == 128) DKZ_TRY(launch_on(stream, name, product_kernel<Tile128, VMC, UMC, false, Epi>, grid, four, g, epi));
            else DKZ_TRY(launch_on(stream, name, product_kernel<Tile64, VMC, UMC, false, Epi>, grid, four, g, epi));
        } else if (p.br == 256) {
            DKZ_TRY(launch_on(stream, name, product_kernel<Tile256, VMC, UMC, true, Epi>, grid, dim3(Tile256::kThreads), g, epi));
        } else if (p.br == 128) {
            DKZ_TRY(launch_on(stream, name, product_kernel<Tile128, VMC, UMC, true, Epi>, grid, four, g, epi));
        } else if (p.bc == 128) {
            DKZ_TRY(launch_on(stream, name, product_kernel<Tile64x128, VMC, UMC, true, Epi>, grid, four, g, epi));
        } else {
            DKZ_TRY(launch_on(stream, name, product_kernel<Tile64, VMC, UMC, true, Epi>, grid, four, g, epi));
        }
    }
    if constexpr (Epi::kElementwise) return join_product(stream, name, g, epi);
    return 0;
}

// The two products of a backward pass, one for the input gradient (u
// row-contiguous) and one for the weights' (both operands), in one launch of one
// kind of tile where that takes less: it saves a launch, and the chip's emptying
// and filling between them. The longer tiles start first. Estimated as the
// longest tile, or all tiles' share of the chip and half a shorter one's for the
// uneven end. Not for products whose K is cut (they fill the chip, 64x4096x4096 is
// 1 us slower paired) nor kinds of which a compute unit holds one (nothing runs
// beside them). A whole backward pass, apart and paired: 64x1024x1024 17.3 and 11.5
// us, 128x4096x1000 18.8 and 13.9, 768x768x3000 31.4 and 25.6, 1536^3 37.2 and 32.4.
// may_cut: the input gradient's K may be cut here too, as it is alone where the rows are few, and how is chosen by what
// is left of the longer tiles when the others have ended (gated blocks, apart, paired as before and so: 200x2048, 2048
// units 38.7, 36.3 and 30.5 us, 512x1024, 4096 units 61.7, 51.2 and 44.4, 333x1001, 1503 units 31.8, 25.9 and 26.2).
inline bool plan_pair(const Product &a, const Product &b, ProductPlan &pa, ProductPlan &pb, bool may_cut = false) {
    const float apart = pa.us + pb.us + kLaunchUs;
    float least = 1e30f;
    bool found = false;
    if ((pa.splits != 1 && !may_cut) || pb.splits != 1 || !a.direct() || !b.direct() || a.rows == 0 || a.cols == 0 || b.rows == 0 || b.cols == 0) return false;
    const uint32_t most = may_cut ? pa.splits : 1;
    for (const TileKind &t : kTileKinds) {
        if (t.occupancy == 1) continue;
        for (uint32_t want = 1; want <= most; ++want) {
            const uint64_t slabs_k = (a.k + 63) / 64, slabs_a = (slabs_k + want - 1) / want, slabs_b = (b.k + 63) / 64;
            const uint64_t splits = slabs_a != 0 ? (slabs_k + slabs_a - 1) / slabs_a : 1;
            const uint64_t tiles_a = splits * div_up(a.rows, t.br) * div_up(a.cols, t.bc), tiles_b = (uint64_t)div_up(b.rows, t.br) * div_up(b.cols, t.bc);
            const uint64_t each = std::min<uint64_t>((tiles_a + tiles_b + kComputeUnits - 1) / kComputeUnits, t.occupancy);
            const float us_a = (float)slabs_a * t.slab[each - 1] + t.fixed, us_b = (float)slabs_b * t.slab[each - 1] + t.fixed;
            const float all = ((float)tiles_a * us_a + (float)tiles_b * us_b) / (float)(kComputeUnits * each);
            // A product's tile takes as long as beside the others of its kind.
            const auto alone = [&](uint64_t slabs, uint64_t tiles) {
                return (float)slabs * t.slab[std::min<uint64_t>((tiles + kComputeUnits - 1) / kComputeUnits, t.occupancy) - 1] + t.fixed;
            };
            const float join = splits > 1 ? join_us(splits, a.rows, a.cols) : 0.0f;
            float us = std::max(std::max(alone(slabs_a, tiles_a), alone(slabs_b, tiles_b)), all + 0.5f * std::min(us_a, us_b));
            if (us + join >= apart || tiles_a + tiles_b > 0x7fffffffull) continue;
            if (may_cut) {  // the longer tiles' slabs that are left, a compute unit's other tiles having ended
                const uint64_t slabs = std::max(slabs_a, slabs_b), tiles = slabs_a > slabs_b ? tiles_a : tiles_b;
                const float left = (float)slabs - all / t.slab[each - 1];
                if (left > 0.0f) us = std::max(us, all + left * t.slab[std::min<uint64_t>((tiles + kComputeUnits - 1) / kComputeUnits, t.occupancy) - 1]);
            }
            us += join;
            if (us >= least) continue;
            least = us;
            pa = {t.br, t.bc, t.wr, t.wc, (uint32_t)splits, (uint32_t)(slabs_a * 64), true, us};
            pb = {t.br, t.bc, t.wr, t.wc, 1, (uint32_t)(slabs_b * 64), true, us};
            found = true;
        }
    }
    return found;
}

// A launch of the two in groups_a + groups_b workgroups.
struct PairLaunch {
    template <class T, class Epi>
    int run(hipStream_t stream, const char *name, const ProductArgs &a, const Epi &epi_a, const ProductArgs &b, const Epi &epi_b, uint32_t groups_a,
            uint32_t groups_b, bool a_first) const {
        return launch_on(stream, name, product_pair_kernel<T, Epi>, dim3(groups_a + groups_b), dim3(T::kThreads), a, epi_a, b, epi_b, groups_a, a_first);
    }
};
template <class T, class Epi, class Pair>
int launch_pair(hipStream_t stream, const char *name, const ProductArgs &a, const Epi &epi_a, const ProductArgs &b, const Epi &epi_b, Pair &pair) {
    DKZ_TRY(pair.template run<T>(stream, name, a, epi_a, b, epi_b, a.tiles_r * a.tiles_c * a.splits, b.tiles_r * b.tiles_c,
                                 std::min(a.k, a.k_chunk) >= b.k));
    return join_product(stream, name, a, epi_a);
}

// The products of a backward pass, each null if it is not wanted; `pair` launches them where they are paired.
template <class Epi, class Pair = PairLaunch>
int run_gradients(hipStream_t stream, const char *name_a, const Product *to_input, const Epi &epi_a, const char *name_b,
                  const Product *to_weights, const Epi &epi_b, float *partial, bool may_cut = false, Pair &&pair = {}) {
    ProductPlan pa{}, pb{};
    if (to_input != nullptr) pa = plan_product(to_input->rows, to_input->cols, to_input->k, false, true, to_input->direct());
    if (to_weights != nullptr) pb = plan_product(to_weights->rows, to_weights->cols, to_weights->k, false, true, to_weights->direct());
    if (to_input == nullptr || to_weights == nullptr || !plan_pair(*to_input, *to_weights, pa, pb, may_cut)) {
        if (to_weights != nullptr) DKZ_TRY((run_product<true, true>(stream, name_b, *to_weights, pb, partial, epi_b)));
        return to_input == nullptr ? 0 : run_product<false, true>(stream, name_a, *to_input, pa, partial, epi_a);
    }
    const Product &a = *to_input, &b = *to_weights;
    const ProductArgs ga = product_args(a, pa, partial), gb = product_args(b, pb, nullptr);
    if (pa.bc == 128) return launch_pair<Tile64x128>(stream, name_a, ga, epi_a, gb, epi_b, pair);
    return launch_pair<Tile64>(stream, name_a, ga, epi_a, gb, epi_b, pair);
}

}  // namespace
}  // namespace dkz
