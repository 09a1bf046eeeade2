// product_f32.hpp -- fp32 products with an epilogue: gemm_split.hpp's kernel (six
// bf16 products on the matrix cores, and the fp32 instruction where those are
// not exact) with partial sums in the caller's workspace.
#pragma once

#include "dense_internal.hpp"
#include "gemm_split.hpp"
#include "gemm_tiling.hpp"

namespace dkz {
namespace {

// Partials of one product at most: 64 MiB, as the library's own products take.
constexpr uint64_t kF32PartialFloats = 1ull << 24;

inline Tiling plan_f32(uint64_t m, uint64_t n, uint64_t k) { return pick_tiling(m, n, k, 1, kF32PartialFloats, false); }

// The bytes of partials that run_f32 takes from the workspace.
inline uint64_t f32_partial_bytes(uint64_t m, uint64_t n, uint64_t k) {
    if (m == 0 || n == 0) return 0;
    const Tiling t = plan_f32(m, n, k);
    if (t.splits > 1) return padded(4 * (uint64_t)t.splits * m * n);
    if (t.stream == 0) return 0;
    const uint64_t tiles = (m + t.bm - 1) / t.bm * ((n + t.bn - 1) / t.bn), rest = tiles - t.full_tiles;
    const uint64_t runs = (rest * ((k + kBK - 1) / kBK) + t.stream - 1) / t.stream;
    return padded(4 * (runs + rest) * t.bm * t.bn);
}

template <Operand AK, Operand BK, class... Epi>
int launch_f32_tiles(hipStream_t stream, const char *name, const Tiling &t, dim3 grid, const SplitArgs &g, const Epi &...epi) {
    const dim3 block(kBlock);
    if (t.bm == 128 && t.bn == 128) return launch_on(stream, name, gemm_split_kernel<128, 128, AK, BK, false, Epi...>, grid, block, g, epi...);
    if (t.bm == 128) return launch_on(stream, name, gemm_split_kernel<128, 64, AK, BK, false, Epi...>, grid, block, g, epi...);
    if (t.bm == 64 && t.bn == 128) return launch_on(stream, name, gemm_split_kernel<64, 128, AK, BK, false, Epi...>, grid, block, g, epi...);
    if (t.bm == 32) return launch_on(stream, name, gemm_split_kernel<32, 128, AK, BK, false, Epi...>, grid, block, g, epi...);
    return launch_on(stream, name, gemm_split_kernel<64, 64, AK, BK, false, Epi...>, grid, block, g, epi...);
}

// C (m x n, leading dimension ldc) = beta * C + op(A) op(B), or every element of the product to `epi`.
// kRowMajor: A is m x k, B n x k; kColMajor: A is k x m, B k x n. `partial` has f32_partial_bytes.
template <Operand AK, Operand BK, class... Epi>
int run_f32(hipStream_t stream, const char *name, const float *a, uint64_t lda, const float *b, uint64_t ldb, float beta, float *c, uint64_t ldc,
            uint64_t m, uint64_t n, uint64_t k, float *partial, const Epi &...epi) {
    if (m == 0 || n == 0) return 0;
    const Tiling t = plan_f32(m, n, k);
    SplitArgs g{};
    g.a = a;
    g.b = b;
    g.c = c;
    g.partial = partial;
    g.m = (uint32_t)m;
    g.n = (uint32_t)n;
    g.k = (uint32_t)k;
    g.lda = (uint32_t)lda;
    g.ldb = (uint32_t)ldb;
    g.ldc = (uint32_t)ldc;
    g.alpha = 1.0f;
    g.beta = beta;
    g.tiles_m = div_up(m, t.bm);
    g.tiles_n = div_up(n, t.bn);
    g.tile_bm = t.bm;
    g.tile_bn_log2 = t.bn == 128 ? 7 : 6;
    g.splits = t.splits;
    g.k_chunk = t.k_chunk;
    uint64_t total = (uint64_t)g.tiles_m * g.tiles_n * g.splits;
    const uint32_t streamed = t.stream ? (uint32_t)(total - t.full_tiles) : 0;
    if (t.stream) {
        const uint32_t slabs = div_up(k, kBK);
        g.full_tiles = t.full_tiles;
        g.stream_len = t.stream;
        g.stream_slabs = streamed * slabs;
        g.div_tile_slabs = make_fastdiv(slabs);
        g.runs = div_up(g.stream_slabs, t.stream);
        total = t.full_tiles + g.runs;
    }
    DKZ_REQUIRE(total <= 0x7fffffffull);
    DKZ_TRY((launch_f32_tiles<AK, BK, Epi...>(stream, name, t, dim3((uint32_t)total), g, epi...)));
    const bool v4 = n % 4 == 0 && ldc % 4 == 0 && aligned16(c);
    const dim3 block(kBlock);
    if (t.stream) {
        const dim3 blocks(streamed * (t.bm * t.bn / 4 / kBlock));
        return v4 ? launch_on(stream, name, stream_reduce_kernel<true, Epi...>, blocks, block, g, epi...)
                  : launch_on(stream, name, stream_reduce_kernel<false, Epi...>, blocks, block, g, epi...);
    }
    if (g.splits == 1) return 0;
    const bool many = g.splits > 32;
    const dim3 blocks(div_up(m * n / (v4 ? 4 : 1), many ? kBlock / 16 : kBlock));
    if (v4)
        return many ? launch_on(stream, name, split_reduce_kernel<true, 16, Epi...>, blocks, block, g, epi...)
                    : launch_on(stream, name, split_reduce_kernel<true, 1, Epi...>, blocks, block, g, epi...);
    return many ? launch_on(stream, name, split_reduce_kernel<false, 16, Epi...>, blocks, block, g, epi...)
                : launch_on(stream, name, split_reduce_kernel<false, 1, Epi...>, blocks, block, g, epi...);
}

}  // namespace
}  // namespace dkz
