// cross_entropy.hip -- softmax cross-entropy of a linear layer over many
// classes without its logits, forward and backward.
//
// Forward, bf16: the product's epilogue reduces every wave's part of a row of
// logits to its maximum m and s = sum of exp(z - m), and a second launch merges
// a row's (m, s) pairs. Backward: the product again, its epilogue making
// d = s_r * (onehot - exp(z - lse)) for a piece of the classes, which the two
// products for the gradients then read. fp32: the logits of a piece are written
// to the workspace and reduced, or replaced by d, there.
#include <algorithm>
#include <type_traits>

#include "dense_internal.hpp"
#include "epilogue.hpp"
#include "product_plan.hpp"
#include "product_f32.hpp"

namespace dkz {
namespace {

__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }

// exp(x) by the exponential instruction: its argument x * log2(e) is rounded in
// fp32, so the result is within |x| * 2^-24 of it, and about 1e-6 for the
// probabilities that matter. NaN in, NaN out.
__device__ __forceinline__ float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }

// The sum s and maximum m of a set of logits, s relative to m: the pair of none is (0, -inf).
struct Stat {
    float m, s;
};
// Merges another set. fmaxf passes over NaNs, which stay in s. A set of -infinities has s 0.
__device__ __forceinline__ Stat merge(Stat a, Stat b) {
    const float m = fmaxf(a.m, b.m);
    const float base = m == neg_inf() ? 0.0f : m;
    return {m, a.s * expf_cw(a.m - base) + b.s * expf_cw(b.m - base)};
}

// A row's results from the pair of all its logits and its target's logit.
__device__ __forceinline__ void finish_row(Stat t, bool target, float z, float *loss, float *lse) {
    // No class left: log(0). A sum that is NaN stays so.
    const float l = t.s == 0.0f ? neg_inf() : t.m + logf(t.s);
    *lse = l;
    // -inf - -inf: the probability 0 of a target among no classes.
    *loss = !target ? 0.0f : l == neg_inf() ? __builtin_inff() : l - z;
}

// ---- bf16 forward ----

struct StatEpilogue {
    static constexpr bool kElementwise = false;
    const float *biases;
    const int *targets;
    Stat *stats;          // [rows][parts]: part = column tile * the workgroup's wave columns + wave column
    float *target_logit;  // [rows]
    uint32_t parts;

    template <int TR, int TC, int WR, int WC>
    __device__ __forceinline__ void tile(const f32x16 (&acc)[TC][TR], uint32_t r0, uint32_t c0, uint32_t wr0, uint32_t wc0,
                                         uint32_t rows, uint32_t cols, uint32_t, uint32_t tc, char *) const {
        constexpr uint32_t kCols = TC * 32;
        const uint32_t lane = threadIdx.x & 63, wave_c = (threadIdx.x >> 6) % WC, first = c0 + wc0;
        const uint32_t cl = first + 4 * (lane >> 5);  // this lane's columns: cl + 8 * n + 0 .. 3
        const auto column = [](int i, int e) { return (uint32_t)(32 * i + 8 * (e >> 2) + (e & 3)); };
        const bool edge = first + kCols > cols;
        // A wave's usual part, inside and without a bias, is taken as it is. (Adding the bias into the accumulators first
        // costs a copy of all 128.)
        const bool plain = biases == nullptr && !edge;
        const auto logit = [&](auto usual, int i, int j, int e) __attribute__((always_inline)) {
            if constexpr (decltype(usual)::value) return acc[i][j][e];
            const uint32_t c = cl + column(i, e);
            return c >= cols ? neg_inf() : biases != nullptr ? acc[i][j][e] + biases[c] : acc[i][j][e];
        };
        const auto part = [&](auto usual, int j) __attribute__((always_inline)) {
            float m = neg_inf();
#pragma unroll
            for (int i = 0; i < TC; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) m = fmaxf(m, logit(usual, i, j, e));
            m = fmaxf(m, __shfl_xor(m, 32));
            const float base = m == neg_inf() ? 0.0f : m;
            float s[2] = {};
#pragma unroll
            for (int i = 0; i < TC; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e & 1] += exp_fast(logit(usual, i, j, e) - base);
            s[0] += s[1];
            return Stat{m, s[0] + __shfl_xor(s[0], 32)};
        };
#pragma unroll
        for (int j = 0; j < TR; ++j) {
            const uint32_t r = r0 + wr0 + 32 * j + (lane & 31);
            const Stat t = plain ? part(std::true_type{}, j) : part(std::false_type{}, j);
            if (r < rows && lane < 32) stats[(uint64_t)r * parts + tc * WC + wave_c] = t;
            // The target's logit, where it is one of this wave's columns: seldom.
            const uint32_t target = r < rows ? (uint32_t)targets[r] : ~0u, o = target - cl;
            if (o < kCols && target < cols && (o & 4) == 0) {
                float z = 0.0f;
#pragma unroll
                for (int i = 0; i < TC; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) z = o == column(i, e) ? acc[i][j][e] : z;
                target_logit[r] = biases != nullptr ? z + biases[target] : z;
            }
        }
    }
    // Few rows: COLS lanes hold a row's part.
    template <int COLS>
    __device__ __forceinline__ void skinny(uint32_t r, uint32_t c, float z, uint32_t rows, uint32_t cols, uint32_t part) const {
        if (c >= cols) z = neg_inf();
        else if (biases != nullptr) z += biases[c];
        if (r < rows && c < cols && c == (uint32_t)targets[r]) target_logit[r] = z;
        const float m = seg_max<COLS>(z), base = m == neg_inf() ? 0.0f : m;
        float s = exp_fast(z - base);
#pragma unroll
        for (int x = 1; x < COLS; x *= 2) s += __shfl_xor(s, x);
        if (r < rows && (threadIdx.x & (COLS - 1)) == 0) stats[(uint64_t)r * parts + part] = {m, s};
    }
};

// Workgroups of the kernels that take a row at a time; beyond, a workgroup takes several.
constexpr uint32_t kRowGroups = 1u << 18;

// A workgroup a row: merges its parts.
__global__ __launch_bounds__(kBlock) void merge_stats_kernel(const Stat *stats, uint32_t parts, const int *targets,
                                                            const float *target_logit, uint32_t rows, uint32_t classes, float *loss,
                                                            float *lse) {
    __shared__ Stat waves[kBlock / kWave];
    for (uint32_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const Stat *row = stats + (uint64_t)r * parts;
        Stat t{neg_inf(), 0.0f};
        for (uint32_t i = threadIdx.x; i < parts; i += 4 * kBlock) {
            Stat next[4];
#pragma unroll
            for (uint32_t u = 0; u < 4; ++u) next[u] = row[min(i + u * kBlock, parts - 1)];
#pragma unroll
            for (uint32_t u = 0; u < 4; ++u)
                if (i + u * kBlock < parts) t = merge(t, next[u]);
        }
#pragma unroll
        for (int x = 1; x < kWave; x *= 2) t = merge(t, {__shfl_xor(t.m, x), __shfl_xor(t.s, x)});
        if (threadIdx.x % kWave == 0) waves[threadIdx.x / kWave] = t;
        __syncthreads();
        if (threadIdx.x == 0) {
#pragma unroll
            for (int w = 1; w < kBlock / kWave; ++w) t = merge(t, waves[w]);
            const bool target = (uint32_t)targets[r] < classes;
            finish_row(t, target, target ? target_logit[r] : 0.0f, loss + r, lse + r);
        }
        __syncthreads();
    }
}

// ---- the gradient of a logit ----

struct RowGradient {
    const int *targets;
    const float *lse, *row_scales;
    float scale;
    uint32_t classes;

    // s_r and lse_r; s_r 0 for a row that has no gradient (then p is not looked at).
    __device__ __forceinline__ void row(uint32_t r, uint32_t &target, float &s, float &l) const {
        target = (uint32_t)targets[r];
        l = lse[r];
        s = row_scales != nullptr ? scale * row_scales[r] : scale;
        if (target >= classes || l == neg_inf()) target = ~0u;
    }
};

// d = s_r * (onehot - exp(z - lse)), rounded to bf16 for the products that read
// it, and each wave's unrounded column sums to `sums` (null: not wanted). The
// tile passes through LDS as TileEpilogue's does.
struct GradientEpilogue {
    static constexpr bool kElementwise = false;
    const float *biases;  // of the piece
    RowGradient rows_of;
    __bf16 *d;            // 16-byte aligned
    uint32_t ldd, first;  // ldd: a multiple of eight; first: the piece's first class
    float *sums;          // [parts of the rows][cols]

    template <int TR, int TC, int WR, int WC>
    __device__ __forceinline__ void tile(const f32x16 (&acc)[TC][TR], uint32_t r0, uint32_t c0, uint32_t wr0, uint32_t wc0,
                                         uint32_t rows, uint32_t cols, uint32_t tr, uint32_t, char *lds) const {
        constexpr uint32_t kCols = TC * 32, kLanes = kCols / 8, kStep = kWave / kLanes, kMask = kCols / 4 - 1;
        const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        float4 *part = reinterpret_cast<float4 *>(lds) + wave * (32 * kCols / 4);
        const uint32_t c = c0 + wc0 + lane % kLanes * 8;
        float bias[8], sum[8] = {};
#pragma unroll
        for (int i = 0; i < 8; ++i) bias[i] = biases != nullptr ? biases[min(c + i, cols - 1)] : 0.0f;
#pragma unroll 1
        for (int j = 0; j < TR; ++j) {
            // Lane x has the values of row x of the 32.
            uint32_t target_of = ~0u;
            float s_of = 0.0f, l_of = 0.0f;
            if (const uint32_t r = r0 + wr0 + 32 * j + (lane & 31); r < rows) rows_of.row(r, target_of, s_of, l_of);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            block_to_lds<TR, TC>(acc, j, part);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll 2
            for (uint32_t x = lane / kLanes; x < 32; x += kStep) {
                const uint32_t r = r0 + wr0 + 32 * j + x, at = x * (kCols / 4), chunk = lane % kLanes * 2;
                const float4 a = part[at + (chunk ^ (x & kMask))], b = part[at + ((chunk + 1) ^ (x & kMask))];
                const uint32_t target = __shfl(target_of, x), hot = target - first - c;
                const float s = __shfl(s_of, x), l = __shfl(l_of, x);
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float p = exp_fast(::dkz::lane(i < 4 ? a : b, i & 3) + bias[i] - l);
                    // NaN logits stay in rows that have a gradient, those past the last class out of it.
                    v[i] = target == ~0u || c + i >= cols ? 0.0f : s * ((hot == (uint32_t)i ? 1.0f : 0.0f) - p);
                    sum[i] += v[i];
                }
                if (r < rows && c < ldd) store8(d, (uint64_t)r * ldd + c, v);
            }
        }
        if (sums == nullptr) return;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
            for (int o = kLanes; o < kWave; o *= 2) sum[i] += __shfl_xor(sum[i], o);
            if (lane < kLanes && c + i < cols) sums[(uint64_t)(tr * WR + wave / WC) * cols + c + i] = sum[i];
        }
    }
    // Few rows: one element, and every row its own part of the sums.
    template <int COLS>
    __device__ __forceinline__ void skinny(uint32_t r, uint32_t c, float z, uint32_t row_count, uint32_t cols, uint32_t) const {
        if (r >= row_count || c >= ldd) return;
        float v = 0.0f;
        uint32_t target;
        float s, l;
        rows_of.row(r, target, s, l);
        if (c < cols && target != ~0u) {
            const float p = exp_fast((biases != nullptr ? z + biases[c] : z) - l);
            v = s * ((target == first + c ? 1.0f : 0.0f) - p);
        }
        store1(d, (uint64_t)r * ldd + c, v);
        if (sums != nullptr && c < cols) sums[(uint64_t)r * cols + c] = v;
    }
};

// ---- fp32 ----

// Logits with their bias, to the workspace.
struct LogitEpilogue : TileEpilogue<LogitEpilogue> {
    const float *biases;
    float *out;
    uint32_t ld;
    LogitEpilogue(const float *biases, float *out, uint64_t ld) : biases(biases), out(out), ld((uint32_t)ld) {}
    __device__ __forceinline__ float bias(uint32_t c) const { return biases != nullptr ? biases[c] : 0.0f; }
    template <int N>
    struct Before {};
    template <int N, class E>
    __device__ __forceinline__ Before<N> before(const E &) const { return {}; }
    template <class E, int N>
    __device__ __forceinline__ void put(const E &e, const float (&bias)[N], float (&z)[N], const Before<N> &) const {
        if (biases != nullptr) {
#pragma unroll
            for (int i = 0; i < N; ++i) z[i] += bias[i];
        }
        store_n(out, e, z);
    }
};

constexpr uint32_t kStatThreads = 512, kStatEach = 8;

// A workgroup a row: the pair of a piece's logits, in one pass with the running
// maximum, merged into the row's; the last piece finishes the row. A thread
// takes eight logits at a time, a workgroup's width apart.
__global__ __launch_bounds__(kStatThreads) void row_stats_kernel(const float *z, uint32_t ld, uint32_t rows, uint32_t cols, uint32_t first,
                                                                uint32_t classes, const int *targets, Stat *run, float *target_logit,
                                                                float *loss, float *lse) {
    __shared__ Stat waves[kStatThreads / kWave];
    for (uint32_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const float *row = z + (uint64_t)r * ld;
        Stat t{neg_inf(), 0.0f};
        for (uint32_t c = threadIdx.x; c < cols; c += kStatEach * kStatThreads) {
            float v[kStatEach], m = t.m;
#pragma unroll
            for (uint32_t i = 0; i < kStatEach; ++i) v[i] = row[min(c + i * kStatThreads, cols - 1)];
#pragma unroll
            for (uint32_t i = 0; i < kStatEach; ++i) m = fmaxf(m, v[i]);
            const float base = m == neg_inf() ? 0.0f : m;
            t.s *= expf_cw(t.m - base);
#pragma unroll
            for (uint32_t i = 0; i < kStatEach; ++i) t.s += c + i * kStatThreads < cols ? expf_cw(v[i] - base) : 0.0f;
            t.m = m;
        }
#pragma unroll
        for (int x = 1; x < kWave; x *= 2) t = merge(t, {__shfl_xor(t.m, x), __shfl_xor(t.s, x)});
        if (threadIdx.x % kWave == 0) waves[threadIdx.x / kWave] = t;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (uint32_t w = 1; w < kStatThreads / kWave; ++w) t = merge(t, waves[w]);
            if (first != 0) t = merge(run[r], t);
            const uint32_t target = (uint32_t)targets[r];
            if (target - first < cols) target_logit[r] = row[target - first];
            run[r] = t;
            if (first + cols == classes)
                finish_row(t, target < classes, target < classes ? target_logit[r] : 0.0f, loss + r, lse + r);
        }
        __syncthreads();
    }
}

constexpr uint32_t kGradRows = 64;  // rows a workgroup of logit_gradient_kernel takes

// A piece's logits become d, and the sums of kGradRows rows' columns go to
// `sums` (null: not). A thread takes four columns of eight rows, its loads
// issued before the first is used; a column's eight threads are added in row
// order. Rows are ld logits long, a multiple of four.
__global__ __launch_bounds__(kBlock) void logit_gradient_kernel(float *z, uint32_t ld, uint32_t rows, uint32_t cols, uint32_t first,
                                                               uint32_t blocks_c, RowGradient rows_of, float *sums) {
    constexpr uint32_t kLanes = 32, kGroups = kBlock / kLanes, kEach = kGradRows / kGroups;
    __shared__ float part[kGroups][kLanes * 4 + 4];
    const uint32_t x = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
    const uint32_t block_r = blockIdx.x / blocks_c, block_c = blockIdx.x - block_r * blocks_c;
    const uint32_t c = (block_c * kLanes + x) * 4, r0 = block_r * kGradRows + group * kEach;
    float4 v[kEach];
    uint32_t target[kEach];
    float s[kEach], l[kEach], sum[4] = {};
    if (c < ld) {
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            const uint32_t r = min(r0 + i, rows - 1);
            v[i] = *reinterpret_cast<const float4 *>(z + (uint64_t)r * ld + c);
            rows_of.row(r, target[i], s[i], l[i]);
        }
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            if (r0 + i >= rows) break;
#pragma unroll
            for (uint32_t w = 0; w < 4; ++w) {
                float &g = ::dkz::lane(v[i], w);
                const float p = expf_cw(g - l[i]);
                g = target[i] == ~0u || c + w >= cols ? 0.0f : s[i] * ((target[i] == first + c + w ? 1.0f : 0.0f) - p);
                sum[w] += g;
            }
            *reinterpret_cast<float4 *>(z + (uint64_t)(r0 + i) * ld + c) = v[i];
        }
    }
    if (sums == nullptr) return;
#pragma unroll
    for (uint32_t w = 0; w < 4; ++w) part[group][x * 4 + w] = sum[w];
    __syncthreads();
    if (threadIdx.x >= kLanes * 4) return;
    float t = part[0][threadIdx.x];
#pragma unroll
    for (uint32_t i = 1; i < kGroups; ++i) t += part[i][threadIdx.x];
    const uint32_t column = block_c * kLanes * 4 + threadIdx.x;
    if (column < cols) sums[(uint64_t)block_r * cols + column] = t;
}

// Rows whose classes are none: lse -infinity, no target, no loss.
__global__ __launch_bounds__(kBlock) void no_classes_kernel(uint32_t rows, float *loss, float *lse) {
    const uint32_t r = blockIdx.x * kBlock + threadIdx.x;
    if (r >= rows) return;
    loss[r] = 0.0f;
    lse[r] = neg_inf();
}

// ---- plans ----

// Bytes of a piece's logits or d where the workspace has room for it: enough rows
// and columns for whole rounds of tiles, and little beside the weights of a class
// count that needs it. A piece has kLeastPiece classes all the same, so that from 2^20
// bf16 rows (2^19 fp32) on it takes more: the products would read all rows' inputs for
// a few columns of tiles each time. bf16's forward pass needs no logits, and no pieces.
constexpr uint64_t kPieceBytes = 512ull << 20;
constexpr uint64_t kLeastPiece = 256;  // classes

// The classes of a piece that fits `bytes` at `per_class` bytes a class, a multiple of 64.
inline uint64_t piece_of(uint64_t classes, uint64_t most_bytes, uint64_t per_class) {
    const uint64_t fit = per_class == 0 ? classes : most_bytes / per_class / 64 * 64;
    return std::min(std::max(fit, kLeastPiece), round_up(classes, 64));
}

struct ForwardPlan {
    uint64_t piece;  // fp32
    uint64_t logits, stats, target, packed, partial;
    uint64_t total() const { return logits + stats + target + packed + partial; }
};
ForwardPlan forward_plan(int type, uint64_t rows, uint64_t inputs, uint64_t classes, uint64_t piece) {
    ForwardPlan p{};
    p.target = padded(4 * rows);
    if (type == DKZ_F32) {
        p.piece = piece;
        p.logits = padded(4 * rows * p.piece);
        p.stats = padded(sizeof(Stat) * rows);
        const uint64_t last = classes % p.piece;
        p.partial = std::max(classes >= p.piece ? f32_partial_bytes(rows, p.piece, inputs) : 0, f32_partial_bytes(rows, last, inputs));
    } else {
        if (!few_rows(rows)) p.packed = packed_bytes(rows, inputs) + packed_bytes(classes, inputs);
        p.stats = padded(sizeof(Stat) * rows * most_of_plans(rows, classes, inputs, true, false, [&](const ProductPlan &t) {
                             return t.row_parts(classes);
                         }));
    }
    return p;
}

struct BackwardPlan {
    uint64_t piece, d, sums, accumulate, packed, partial;
    uint64_t total() const { return d + sums + accumulate + packed + partial; }
};
BackwardPlan backward_plan(int type, uint64_t rows, uint64_t inputs, uint64_t classes, uint64_t piece) {
    BackwardPlan p{};
    const uint64_t size = type_size(type);
    p.piece = piece;
    p.d = padded(size * rows * p.piece);
    const uint64_t last = classes % p.piece, whole = classes >= p.piece ? p.piece : 0;
    if (type == DKZ_F32) {
        p.sums = padded(4 * p.piece * div_up(rows, kGradRows));
        for (const uint64_t n : {whole, last}) {
            if (n == 0) continue;
            p.partial = std::max({p.partial, f32_partial_bytes(rows, n, inputs), f32_partial_bytes(n, inputs, rows),
                                  f32_partial_bytes(rows, inputs, n)});
        }
    } else {
        if (rows != 0) p.packed = packed_bytes(rows, inputs) + packed_bytes(classes, inputs);
        // The input gradient of several pieces is summed in fp32.
        if (classes > p.piece) p.accumulate = padded(4 * rows * inputs);
        for (const uint64_t n : {whole, last}) {
            if (n == 0) continue;
            p.sums = std::max(p.sums, padded(4 * n * most_of_plans(rows, n, inputs, true, false, [&](const ProductPlan &t) {
                                                 return t.column_parts(rows);
                                             })));
            p.partial = std::max({p.partial, most_partial_bytes(n, inputs, rows, false), most_partial_bytes(rows, inputs, n, false)});
        }
    }
    return p;
}

// Calls f with the plans of pieces of at most kPieceBytes, half of that, and so on, the largest first, until it returns
// true; whether it did. Most halvings leave a piece as it is, bounded at both ends: each piece is planned once, as planning
// costs the host microseconds (1x432x8493 fp32: all 31 halvings 60 us, the first plan 4).
template <class Plan, class F>
bool each_plan(Plan (*make)(int, uint64_t, uint64_t, uint64_t, uint64_t), int type, uint64_t rows, uint64_t inputs, uint64_t classes, F f) {
    uint64_t last = ~0ull;
    for (uint64_t most = kPieceBytes;; most /= 2) {
        const uint64_t piece = piece_of(classes, most, type_size(type) * rows);
        if (piece != last && f(make(type, rows, inputs, classes, piece))) return true;
        if (most == 0) return false;
        last = piece;
    }
}

// The first of these plans that `bytes` has room for.
template <class Plan>
bool fit_plan(Plan (*make)(int, uint64_t, uint64_t, uint64_t, uint64_t), int type, uint64_t rows, uint64_t inputs, uint64_t classes,
              uint64_t bytes, Plan &plan) {
    return each_plan(make, type, rows, inputs, classes, [&](const Plan &p) {
        plan = p;
        return p.total() <= bytes;
    });
}

// The bytes of the smallest of these plans (not always the one with the smallest pieces: one piece needs no fp32 sums of
// the input gradient), and of the first.
template <class Plan>
void plan_bytes(Plan (*make)(int, uint64_t, uint64_t, uint64_t, uint64_t), int type, uint64_t rows, uint64_t inputs, uint64_t classes,
                size_t *least, size_t *best) {
    *least = *best = 0;
    each_plan(make, type, rows, inputs, classes, [&](const Plan &p) {
        if (*best == 0) *least = *best = (size_t)p.total();
        *least = std::min(*least, (size_t)p.total());
        return false;
    });
}

// The input gradient of one of several pieces: added up in fp32, the last one rounded to out.
struct PieceEpilogue : TileEpilogue<PieceEpilogue> {
    float *sum;
    __bf16 *out;  // null but for the last piece
    uint32_t ld;
    bool begin, words;
    __device__ __forceinline__ float bias(uint32_t) const { return 0.0f; }
    __device__ __forceinline__ bool in_words() const { return words; }
    template <int N>
    using Before = Raw<float, N>;
    template <int N, class E>
    __device__ __forceinline__ Before<N> before(const E &e) const {
        Before<N> o = {};
        if (!begin) load_raw<float, E, N>(sum, e, o);
        return o;
    }
    template <class E, int N>
    __device__ __forceinline__ void put(const E &e, const float (&)[N], float (&z)[N], const Before<N> &o) const {
        if (!begin) {
#pragma unroll
            for (int i = 0; i < N; ++i) z[i] += o[i];
        }
        if (out != nullptr) store_n(out, e, z);
        else store_n(sum, e, z);
    }
};

int forward(hipStream_t stream, int type, uint64_t rows, uint64_t inputs, uint64_t classes, const void *input, const void *weights,
            const float *biases, const int *targets, float *loss, float *lse, const ForwardPlan &plan, Workspace ws) {
    constexpr const char *kName = "linear_cross_entropy";
    if (classes == 0)
        return launch_on(stream, "linear_cross_entropy_none", no_classes_kernel, dim3(div_up(rows, kBlock)), dim3(kBlock), (uint32_t)rows, loss, lse);
    float *target_logit = ws.take<float>(plan.target / 4);
    Stat *stats = ws.take<Stat>(plan.stats / sizeof(Stat));
    if (type == DKZ_BF16) {
        Matrix x{static_cast<const __bf16 *>(input), inputs}, w{static_cast<const __bf16 *>(weights), inputs};
        if (!few_rows(rows)) DKZ_TRY(pack(stream, x, rows, w, classes, inputs, ws));
        const ProductPlan p = plan_product(rows, classes, inputs, true, false, operands_direct(x.p, x.ld, w.p, w.ld));
        const uint32_t parts = (uint32_t)p.row_parts(classes);
        const StatEpilogue epi{biases, targets, stats, target_logit, parts};
        DKZ_TRY((run_product<false, false>(stream, kName, {x.p, x.ld, w.p, w.ld, rows, classes, inputs}, p, nullptr, epi)));
        return launch_on(stream, "linear_cross_entropy_merge", merge_stats_kernel, dim3(std::min((uint32_t)rows, kRowGroups)), dim3(kBlock), stats,
                      parts, targets, target_logit, (uint32_t)rows, (uint32_t)classes, loss, lse);
    }
    float *logits = ws.take<float>(plan.logits / 4), *partial = ws.take<float>(plan.partial / 4);
    for (uint64_t first = 0; first < classes; first += plan.piece) {
        const uint64_t n = std::min(plan.piece, classes - first), ld = round_up(n, 4);
        const LogitEpilogue epi(biases != nullptr ? biases + first : nullptr, logits, ld);
        DKZ_TRY((run_f32<kRowMajor, kRowMajor>(stream, kName, static_cast<const float *>(input), inputs,
                                               static_cast<const float *>(weights) + first * inputs, inputs, 0.0f, (float *)nullptr, ld,
                                               rows, n, inputs, partial, epi)));
        DKZ_TRY(launch_on(stream, "linear_cross_entropy_stats", row_stats_kernel, dim3(std::min((uint32_t)rows, kRowGroups)),
                          dim3(kStatThreads), logits, (uint32_t)ld, (uint32_t)rows, (uint32_t)n, (uint32_t)first, (uint32_t)classes, targets,
                          stats, target_logit, loss, lse));
    }
    return 0;
}

constexpr const char *kWeights = "linear_cross_entropy_weights", *kInput = "linear_cross_entropy_input";

int backward_f32(hipStream_t stream, uint64_t rows, uint64_t inputs, uint64_t classes, const float *input, const float *weights, const float *biases,
                 const RowGradient &grad, float beta, float *bias_updates, float *weight_updates, float *input_delta,
                 const BackwardPlan &plan, Workspace ws) {
    float *d = ws.take<float>(plan.d / 4), *sums = ws.take<float>(plan.sums / 4), *partial = ws.take<float>(plan.partial / 4);
    for (uint64_t first = 0; first < classes; first += plan.piece) {
        const uint64_t n = std::min(plan.piece, classes - first), ld = round_up(n, 4), chunks = div_up(rows, kGradRows);
        const float *w = weights + first * inputs;
        if (rows != 0) {
            const LogitEpilogue epi(biases != nullptr ? biases + first : nullptr, d, ld);
            DKZ_TRY((run_f32<kRowMajor, kRowMajor>(stream, "linear_cross_entropy_logits", input, inputs, w, inputs, 0.0f, (float *)nullptr, ld, rows,
                                                   n, inputs, partial, epi)));
            DKZ_TRY(launch_on(stream, "linear_cross_entropy_gradient", logit_gradient_kernel, dim3(div_up(ld, 128) * (uint32_t)chunks), dim3(kBlock),
                              d, (uint32_t)ld, (uint32_t)rows, (uint32_t)n, (uint32_t)first, div_up(ld, 128), grad,
                              bias_updates != nullptr ? sums : nullptr));
        }
        if (bias_updates != nullptr) DKZ_TRY(add_column_sums(stream, sums, chunks, n, beta, bias_updates + first));
        if (weight_updates != nullptr)
            DKZ_TRY((run_f32<kColMajor, kColMajor>(stream, kWeights, d, ld, input, inputs, beta, weight_updates + first * inputs, inputs, n, inputs,
                                                   rows, partial)));
        if (input_delta != nullptr)
            DKZ_TRY((run_f32<kRowMajor, kColMajor>(stream, kInput, d, ld, w, inputs, first == 0 ? 0.0f : 1.0f, input_delta, inputs, rows, inputs, n,
                                                   partial)));
    }
    return 0;
}

int backward_bf16(hipStream_t stream, uint64_t rows, uint64_t inputs, uint64_t classes, const __bf16 *input, const __bf16 *weights,
                  const float *biases, const RowGradient &grad, float beta, float *bias_updates, __bf16 *weight_updates,
                  __bf16 *input_delta, const BackwardPlan &plan, Workspace ws) {
    __bf16 *d = ws.take<__bf16>(plan.d / 2);
    float *sums = ws.take<float>(plan.sums / 4), *accumulate = ws.take<float>(plan.accumulate / 4);
    float *partial = ws.take<float>(plan.partial / 4);
    Matrix x{input, inputs}, all{weights, inputs};
    if (rows != 0) DKZ_TRY(pack(stream, x, rows, all, classes, inputs, ws));
    for (uint64_t first = 0; first < classes; first += plan.piece) {
        const __bf16 *w = all.p + first * all.ld;
        const uint64_t n = std::min(plan.piece, classes - first), ldd = round_up(n, 8);
        const ProductPlan p =
            plan_product(rows, n, inputs, true, false, operands_direct(x.p, x.ld, w, all.ld));
        const uint64_t chunks = p.column_parts(rows);
        const GradientEpilogue epi{biases != nullptr ? biases + first : nullptr, grad, d, (uint32_t)ldd, (uint32_t)first,
                                            bias_updates != nullptr ? sums : nullptr};
        DKZ_TRY((run_product<false, false>(stream, "linear_cross_entropy_gradient", {x.p, x.ld, w, all.ld, rows, n, inputs}, p, nullptr, epi)));
        if (bias_updates != nullptr) DKZ_TRY(add_column_sums(stream, sums, chunks, n, beta, bias_updates + first));
        const Product to_input{d, ldd, w, all.ld, rows, inputs, n}, to_weights{d, ldd, x.p, x.ld, n, inputs, rows};
        __bf16 *updates = weight_updates != nullptr ? weight_updates + first * inputs : nullptr;
        const auto epi_weights = store_epilogue<__bf16>(updates, nullptr, inputs, beta);
        const bool one = n == classes;
        DKZ_TRY(run_gradients(stream, kInput, one && input_delta != nullptr ? &to_input : nullptr,
                              store_epilogue<__bf16>(input_delta, nullptr, inputs, 0.0f), kWeights, updates != nullptr ? &to_weights : nullptr, epi_weights, partial));
        if (!one && input_delta != nullptr) {
            PieceEpilogue e;
            e.sum = accumulate;
            e.out = first + n == classes ? input_delta : nullptr;
            e.ld = (uint32_t)inputs;
            e.begin = first == 0;
            e.words = e.out == nullptr || rows_in_words<__bf16>(inputs, e.out);
            DKZ_TRY((run_product<false, true>(stream, kInput, to_input, plan_product(rows, inputs, n, false, true, to_input.direct()), partial, e)));
        }
    }
    return 0;
}

}  // namespace
}  // namespace dkz

using namespace dkz;

extern "C" {

int dkz_linear_cross_entropy_forward_workspace(int type, int rows, int inputs, int classes, size_t *least, size_t *best) {
    DKZ_REQUIRE(least != nullptr && best != nullptr && type_ok(type) && rows >= 0 && inputs >= 0 && classes >= 0);
    DKZ_REQUIRE_SIDE(rows);
    DKZ_REQUIRE_SIDE(inputs);
    DKZ_REQUIRE_SIDE(classes);
    DKZ_REQUIRE((uint64_t)rows * (uint64_t)classes <= 1ull << 38);
    DKZ_REQUIRE_ELEMS(rows, inputs);
    DKZ_REQUIRE_ELEMS(classes, inputs);
    const uint64_t m = (uint64_t)rows, k = (uint64_t)inputs, n = (uint64_t)classes;
    *least = *best = 0;
    if (m != 0 && n != 0) plan_bytes(forward_plan, type, m, k, n, least, best);
    return 0;
}

int dkz_linear_cross_entropy_forward(int type, int rows, int inputs, int classes, const void *input, const void *weights,
                                     const float *biases, const int *targets, float *loss, float *lse, void *workspace,
                                     size_t workspace_bytes) {
    DKZ_REQUIRE(type_ok(type) && rows >= 0 && inputs >= 0 && classes >= 0);
    DKZ_REQUIRE_SIDE(rows);
    DKZ_REQUIRE_SIDE(inputs);
    DKZ_REQUIRE_SIDE(classes);
    DKZ_REQUIRE((uint64_t)rows * (uint64_t)classes <= 1ull << 38);
    DKZ_REQUIRE_ELEMS(rows, inputs);
    DKZ_REQUIRE_ELEMS(classes, inputs);
    if (rows == 0) return 0;
    DKZ_REQUIRE(targets != nullptr && loss != nullptr && lse != nullptr);
    DKZ_REQUIRE(inputs == 0 || classes == 0 || (input != nullptr && weights != nullptr));
    const uint64_t m = (uint64_t)rows, k = (uint64_t)inputs, n = (uint64_t)classes, size = type_size(type);
    ForwardPlan plan{};
    if (n != 0) {
        DKZ_REQUIRE(workspace != nullptr && aligned16(workspace));
        DKZ_REQUIRE(fit_plan(forward_plan, type, m, k, n, workspace_bytes, plan));
    }
    const Span writes[] = {{loss, 4 * m}, {lse, 4 * m}, {workspace, plan.total()}};
    const Span reads[] = {{input, m * k * size}, {weights, n * k * size}, {biases, 4 * n}, {targets, 4 * m}};
    DKZ_REQUIRE(disjoint(writes, reads));
    return forward(current_stream(), type, m, k, n, input, weights, biases, targets, loss, lse, plan, {static_cast<char *>(workspace), plan.total()});
}

int dkz_linear_cross_entropy_backward_workspace(int type, int rows, int inputs, int classes, size_t *least, size_t *best) {
    DKZ_REQUIRE(least != nullptr && best != nullptr && type_ok(type) && rows >= 0 && inputs >= 0 && classes >= 0);
    DKZ_REQUIRE_SIDE(rows);
    DKZ_REQUIRE_SIDE(inputs);
    DKZ_REQUIRE_SIDE(classes);
    DKZ_REQUIRE((uint64_t)rows * (uint64_t)classes <= 1ull << 38);
    DKZ_REQUIRE_ELEMS(rows, inputs);
    DKZ_REQUIRE_ELEMS(classes, inputs);
    const uint64_t m = (uint64_t)rows, k = (uint64_t)inputs, n = (uint64_t)classes;
    *least = *best = 0;
    if (n != 0) plan_bytes(backward_plan, type, m, k, n, least, best);
    return 0;
}

int dkz_linear_cross_entropy_backward(int type, int rows, int inputs, int classes, const void *input, const void *weights,
                                      const float *biases, const int *targets, const float *lse, const float *row_scales,
                                      float scale, float beta, float *bias_updates, void *weight_updates, void *input_delta,
                                      void *workspace, size_t workspace_bytes) {
    DKZ_REQUIRE(type_ok(type) && rows >= 0 && inputs >= 0 && classes >= 0);
    DKZ_REQUIRE_SIDE(rows);
    DKZ_REQUIRE_SIDE(inputs);
    DKZ_REQUIRE_SIDE(classes);
    DKZ_REQUIRE((uint64_t)rows * (uint64_t)classes <= 1ull << 38);
    DKZ_REQUIRE_ELEMS(rows, inputs);
    DKZ_REQUIRE_ELEMS(classes, inputs);
    const uint64_t m = (uint64_t)rows, k = (uint64_t)inputs, n = (uint64_t)classes, size = type_size(type);
    if (bias_updates == nullptr && weight_updates == nullptr && input_delta == nullptr) return 0;
    if (m != 0 && n != 0) {
        DKZ_REQUIRE(targets != nullptr && lse != nullptr);
        DKZ_REQUIRE(k == 0 || (input != nullptr && weights != nullptr));
    }
    BackwardPlan plan{};
    if (n != 0) {
        DKZ_REQUIRE(fit_plan(backward_plan, type, m, k, n, workspace_bytes, plan));
        DKZ_REQUIRE(plan.total() == 0 || (workspace != nullptr && aligned16(workspace)));
    }
    const Span writes[] = {{bias_updates, 4 * n}, {weight_updates, n * k * size}, {input_delta, m * k * size}, {workspace, plan.total()}};
    const Span reads[] = {{input, m * k * size}, {weights, n * k * size}, {biases, 4 * n}, {targets, 4 * m}, {lse, 4 * m}, {row_scales, 4 * m}};
    DKZ_REQUIRE(disjoint(writes, reads));
    const RowGradient grad{targets, lse, row_scales, scale, (uint32_t)n};
    const Workspace ws{static_cast<char *>(workspace), plan.total()};
    const hipStream_t stream = current_stream();
    if (n == 0) {  // no class pulls at the input
        if (input_delta == nullptr || m * k == 0) return 0;
        if (type == DKZ_F32)
            return run_f32<kRowMajor, kColMajor>(stream, kInput, (const float *)nullptr, 0, (const float *)nullptr, k, 0.0f,
                                                 static_cast<float *>(input_delta), k, m, k, 0, nullptr);
        return run_product<false, true>(stream, kInput, {nullptr, 0, nullptr, k, m, k, 0}, plan_product(m, k, 0, false, false, true), nullptr,
                                        store_epilogue<__bf16>(input_delta, nullptr, k, 0.0f));
    }
    if (type == DKZ_F32)
        return backward_f32(stream, m, k, n, static_cast<const float *>(input), static_cast<const float *>(weights), biases, grad, beta,
                            bias_updates, static_cast<float *>(weight_updates), static_cast<float *>(input_delta), plan, ws);
    return backward_bf16(stream, m, k, n, static_cast<const __bf16 *>(input), static_cast<const __bf16 *>(weights), biases, grad, beta, bias_updates,
                         static_cast<__bf16 *>(weight_updates), static_cast<__bf16 *>(input_delta), plan, ws);
}

}  // extern "C"
