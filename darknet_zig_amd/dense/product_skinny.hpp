// product_skinny.hpp -- bf16 products of few rows (a token, a handful of
// sequences): every weight is read once and used for a few rows, so the time is
// the weights' way from memory.
//
// A workgroup takes 16 * CT columns and all rows, its waves a share of K each:
// no LDS on the way, a lane loads eight k of a weight row straight into an operand
// of v_mfma_f32_16x16x32_bf16 and eight of an input row, which the caches hold,
// into the other. Each wave keeps two or four steps of 64 k in flight. The waves'
// sums meet in LDS in wave order, and the epilogue takes them from there. One row
// of 4096 to 16384 outputs 25.1 us (5.3 TB/s), 32768 47.4 (5.7), 4096 8.5; with weights
// that the caches hold 21.3, 39.7 and 6.9.
#pragma once

#include "dense_internal.hpp"
#include "product.hpp"

namespace dkz {
namespace {

typedef short s16x8w __attribute__((ext_vector_type(8), aligned(4)));
typedef float f32x4v __attribute__((ext_vector_type(4)));

// Rows at most: 4096x4096 weights in the caches take 6.9 us at one row, 9.6 at 16 and
// 13.3 at 32, where tiles take 13.6 (at 64 they take no more, this kernel 20.4).
constexpr uint32_t kSkinnyRows = 32;
constexpr int kSkinnyWaves = 4;
inline bool few_rows(uint64_t rows) { return rows <= kSkinnyRows; }

// ODD: rows may start inside a 4-byte word.
template <int RT, int CT, bool ODD, class Epi>
__global__ __launch_bounds__(64 * kSkinnyWaves) void skinny_kernel(ProductArgs g, Epi epi) {
    constexpr int kCols = 16 * CT, kRows = 16 * RT, kPitch = kCols + 4, kWaves = kSkinnyWaves;
    __shared__ __align__(16) float sums[kWaves][kRows][kPitch];
    // In a scalar, so that what depends on it is a branch: matrix instructions take no notice of masked lanes.
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t lane = threadIdx.x & 63, l16 = lane & 15, group = lane >> 4;
    // Pairs go in the workgroups' own order: a front of each half moves through memory. (In runs, sixteen fronts whose distances
    // are powers of two where the sizes are: 1x4096, 8192 units from memory 31.1 us, 25.2 so; 16384 units 58.2 and 48.2.)
    const uint32_t c0 = (kPaired<Epi> ? blockIdx.x : xcd_run(blockIdx.x, gridDim.x)) * kCols;
    // This wave's K: whole steps of 64 but for the last wave's end.
    const uint32_t steps = (g.k + 63) / 64, per = (steps + kWaves - 1) / kWaves;
    const uint32_t first = min(wave * per, steps), last = min(first + per, steps);

    f32x4v acc[CT][RT] = {};
    const short *pu[CT], *pv[RT];
#pragma unroll
    for (int i = 0; i < CT; ++i) {  // columns past the end repeat the last one, rows the last row: not stored
        uint32_t row = min(c0 + 16 * i + l16, g.cols - 1);
        if constexpr (kPaired<Epi>) row = min(Pairs::row(row, epi.half), 2 * epi.half - 1);
        pu[i] = reinterpret_cast<const short *>(g.u) + (uint64_t)row * g.ldu + 16 * group;
    }
#pragma unroll
    for (int j = 0; j < RT; ++j)
        pv[j] = reinterpret_cast<const short *>(g.v) + (uint64_t)min(16 * j + l16, g.rows - 1) * g.ldv + 16 * group;

    // A step's k 16 * group + 0 .. 15 of a row, in two operands: both sides name the same k by the same lane and place.
    struct Step {
        s16x8 u[CT][2], v[RT][2];
    };
    auto eight = [&](const short *p) __attribute__((always_inline)) {
        if constexpr (ODD) return load_shifted(p);
        else return (s16x8)*reinterpret_cast<const s16x8w *>(p);
    };
    auto load = [&](Step &s, uint32_t step) __attribute__((always_inline)) {
        const uint32_t k = step * 64;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < CT; ++i) s.u[i][h] = eight(pu[i] + k + 8 * h);
#pragma unroll
            for (int j = 0; j < RT; ++j) s.v[j][h] = eight(pv[j] + k + 8 * h);
        }
    };
    auto load_end = [&](Step &s, uint32_t step) __attribute__((always_inline)) {  // k past the end read as 0
        const uint32_t k = step * 64 + 16 * group;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                const bool in = k + 8 * h + x < g.k;
#pragma unroll
                for (int i = 0; i < CT; ++i) s.u[i][h][x] = in ? pu[i][step * 64 + 8 * h + x] : (short)0;
#pragma unroll
                for (int j = 0; j < RT; ++j) s.v[j][h][x] = in ? pv[j][step * 64 + 8 * h + x] : (short)0;
            }
    };
    auto multiply = [&](const Step &s) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < CT; ++i)
#pragma unroll
                for (int j = 0; j < RT; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, s.u[i][h]),
                                                                       __builtin_bit_cast(bf16x8, s.v[j][h]), acc[i][j], 0, 0, 0);
    };
    const bool ragged = last == steps && first < last && g.k % 64 != 0;
    const uint32_t whole = last - ragged;
    if (first < whole) {
        constexpr uint32_t kAhead = RT * CT >= 4 ? 2 : 4;  // steps in flight
        Step s[kAhead];
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a)
            if (first + a < whole) load(s[a], first + a);
        uint32_t step = first;
#pragma unroll 1
        for (; step + 2 * kAhead <= whole; step += kAhead) {
#pragma unroll
            for (uint32_t a = 0; a < kAhead; ++a) {
                multiply(s[a]);
                load(s[a], step + a + kAhead);
            }
        }
        // Fewer than two rounds are left.
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a) {
            if (step + a < whole) multiply(s[a]);
            if (step + a + kAhead < whole) load(s[a], step + a + kAhead);
        }
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a)
            if (step + a + kAhead < whole) multiply(s[a]);
    }
    if (ragged) {
        Step s;
        load_end(s, whole);
        multiply(s);
    }
    // acc[i][j][e] is column 16 * i + 4 * group + e of row 16 * j + l16.
#pragma unroll
    for (int i = 0; i < CT; ++i)
#pragma unroll
        for (int j = 0; j < RT; ++j)
            *reinterpret_cast<f32x4v *>(&sums[wave][16 * j + l16][16 * i + 4 * group]) = acc[i][j];
    __syncthreads();
    if constexpr (kPaired<Epi>) {
        // A thread a pair.
        for (uint32_t e = threadIdx.x; e < kRows * kCols / 2; e += 64 * kWaves) {
            const uint32_t r = e / (kCols / 2), j = e % (kCols / 2), c = j / 8 * 16 + j % 8;
            float x = sums[0][r][c], y = sums[0][r][c + 8];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) {
                x += sums[w][r][c];
                y += sums[w][r][c + 8];
            }
            epi.pair(r, c0 / 2 + j, x, y, g.rows);
        }
        return;
    }
    // A thread an element, the columns along the lanes.
    for (uint32_t e = threadIdx.x; e < kRows * kCols; e += 64 * kWaves) {
        const uint32_t r = e / kCols, c = e % kCols;
        float z = sums[0][r][c];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) z += sums[w][r][c];
        if constexpr (!kPaired<Epi>) epi.template skinny<kCols>(r, c0 + c, z, g.rows, g.cols, c0 / kCols);
    }
}

// Columns of a workgroup, 16 or 32. (Eight waves and 16 columns take as long as four
// or, 1x16384x4096, a third longer.) Up to 16 rows: what gives the compute
// units as many workgroups each, as far as it can, 32 where both do; but 16 where K
// is long (us for 32 and 16 columns at K 4096: 8192 columns 13.6 and 15.0, 18432
// 31.4 and 26.7, 24576 35.6 and 38.7; 8192x8192 30.9 and 28.4). More rows: 32 unless
// that leaves compute units without (20 rows, K 4096: 4096 columns 16.4 and 12.3, 6144
// 16.6 and 21.1, 16384 32.0 and 43.1).
inline uint32_t skinny_columns(uint64_t rows, uint64_t cols, uint64_t k) {
    constexpr uint64_t kUnits = 256;
    if (rows > 16) return cols > 16 * kUnits ? 32 : 16;
    const auto rounded = [&](uint64_t width) { return round_up((cols + width - 1) / width, kUnits) * width; };
    return k < 8192 && rounded(32) <= rounded(16) ? 32 : 16;
}

template <int RT, int CT, class Epi>
int launch_skinny(hipStream_t stream, const char *name, dim3 grid, const ProductArgs &g, const Epi &epi) {
    const bool odd = ((g.ldv | g.ldu) & 1) != 0 || (((uintptr_t)g.v | (uintptr_t)g.u) & 3) != 0;
    if (odd) return launch_on(stream, name, skinny_kernel<RT, CT, true, Epi>, grid, dim3(64 * kSkinnyWaves), g, epi);
    return launch_on(stream, name, skinny_kernel<RT, CT, false, Epi>, grid, dim3(64 * kSkinnyWaves), g, epi);
}

template <class Epi>
int run_skinny(hipStream_t stream, const char *name, const __bf16 *v, uint64_t ldv, const __bf16 *u, uint64_t ldu, uint64_t rows,
               uint64_t cols, uint64_t k, uint32_t width, const Epi &epi) {
    ProductArgs g{};
    g.v = v;
    g.u = u;
    g.ldv = (uint32_t)ldv;
    g.ldu = (uint32_t)ldu;
    g.rows = (uint32_t)rows;
    g.cols = (uint32_t)cols;
    g.k = (uint32_t)k;
    const dim3 grid(div_up(cols, width));
    if (rows <= 16) return width == 32 ? launch_skinny<1, 2>(stream, name, grid, g, epi) : launch_skinny<1, 1>(stream, name, grid, g, epi);
    return width == 32 ? launch_skinny<2, 2>(stream, name, grid, g, epi) : launch_skinny<2, 1>(stream, name, grid, g, epi);
}

}  // namespace
}  // namespace dkz
