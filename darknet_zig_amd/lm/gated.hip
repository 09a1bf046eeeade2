// gated.hip -- a gated feed-forward block: both projections, the gate's activation
// and the product of the two, and its backward pass.
//
// bf16: one product whose columns come in pairs of the two halves (kPaired), so that
// the epilogue finds a unit's gate and its other projection in one lane. Backward: one
// pass over the kept projections makes d, as [rows, 2 * hidden], and the two products
// of a linear layer follow. fp32: the split product writes the projections, and a
// second pass makes the output.
#include <utility>

#include "dense_internal.hpp"
#include "dkz_lm.h"
#include "epilogue.hpp"
#include "product_f32.hpp"
#include "product_plan.hpp"

namespace dkz {
namespace {

// ---- the gate ----

// u = g * (one + three * g^2), and the activation g * logistic(u), or logistic(u)
// alone. (g^2 is bounded, so that 0 * g^2 is 0.)
struct Gate {
    float one, three;
    bool alone, relu;

    __device__ __forceinline__ float inner(float g) const { return g * (one + three * fminf(g * g, 1e30f)); }
    __device__ __forceinline__ float slope(float g) const { return one + 3.0f * three * fminf(g * g, 1e30f); }
};

inline bool gate_ok(int a) { return a == DKZ_LOGISTIC || a == DKZ_RELU || a == DKZ_LINEAR || a == DKZ_SILU || a == DKZ_GELU; }
inline bool gate_has_exp(int a) { return a != DKZ_RELU && a != DKZ_LINEAR; }
inline Gate make_gate(int a) {
    const float c = 1.59576912160573071f;  // 2 * sqrt(2 / pi): (1 + tanh(x)) / 2 is logistic(2 * x)
    return a == DKZ_GELU ? Gate{c, c * 0.044715f, false, false} : Gate{1.0f, 0.0f, a == DKZ_LOGISTIC, a == DKZ_RELU};
}

// logistic(u) for a result of type T. bf16: the exponential and reciprocal instructions, together within (|u| + 2) * 2^-23
// of it, which is below 2^-16 where it is above 2^-128.
template <class T>
__device__ __forceinline__ float logistic(float u) {
    if constexpr (sizeof(T) == 2) return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(u * -1.44269504088896341f));
    else return 1.0f / (1.0f + expf_cw(-u));
}

// The activation at g. EXP: one with a logistic.
template <class T, bool EXP>
__device__ __forceinline__ float activate_gate(const Gate &gate, float g) {
    if constexpr (EXP) {
        const float p = logistic<T>(gate.inner(g));
        return gate.alone ? p : g * p;
    } else {
        return gate.relu && !(g > 0.0f) ? (g != g ? g : 0.0f) : g;
    }
}
// It and its derivative.
template <class T, bool EXP>
__device__ __forceinline__ float gate_slope(const Gate &gate, float g, float &a) {
    if constexpr (EXP) {
        const float u = gate.inner(g), p = logistic<T>(u), rest = logistic<T>(-u), curve = p * rest;
        a = gate.alone ? p : g * p;
        return gate.alone ? curve : p + g * (curve * gate.slope(g));
    } else {
        const bool on = !gate.relu || g > 0.0f;
        a = on ? g : g != g ? g : 0.0f;
        return on ? 1.0f : 0.0f;
    }
}

// ---- forward ----

// output(r, j) = activation(s(r, j)) * s(r, half + j), and s itself to `sums` if it is wanted.
template <class T, bool EXP>
struct GatedEpilogue {
    static constexpr bool kElementwise = false;  // its pieces are joined in pairs
    const float *biases;
    T *sums, *output;
    uint32_t half;
    Gate gate;

    // Units j .. j + N - 1 of row r, n of them there.
    template <int N>
    __device__ __forceinline__ void put(uint32_t r, uint32_t j, uint32_t n, float (&x)[N], float (&y)[N]) const {
        if (sums != nullptr) {
            const uint64_t at = (uint64_t)r * 2 * half + j;
            store_n(sums, RowRun{at, n}, x);
            store_n(sums, RowRun{at + half, n}, y);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = activate_gate<T, EXP>(gate, x[i]) * y[i];
        store_n(output, RowRun{(uint64_t)r * half + j, n}, x);
    }
    template <int N>
    __device__ __forceinline__ void add_bias(uint32_t j, float (&x)[N], float (&y)[N]) const {
        if (biases == nullptr) return;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t c = min(j + i, half - 1);
            x[i] += biases[c];
            y[i] += biases[half + c];
        }
    }
    // Few rows: one unit, if it is there.
    __device__ __forceinline__ void pair(uint32_t r, uint32_t j, float x, float y, uint32_t rows) const {
        if (r >= rows || j >= half) return;
        float a[1] = {x}, b[1] = {y};
        add_bias(j, a, b);
        put(r, j, 1, a, b);
    }
    // A lane takes sixteen columns of a row, eight units.
    template <int TR, int TC, int WR, int WC>
    __device__ __forceinline__ void tile(const f32x16 (&acc)[TC][TR], uint32_t r0, uint32_t c0, uint32_t wr0, uint32_t wc0,
                                         uint32_t rows, uint32_t, uint32_t, uint32_t, char *lds) const {
        constexpr uint32_t kCols = TC * 32, kLanes = kCols / 16, kStep = kWave / kLanes, kMask = kCols / 4 - 1;
        const uint32_t lane = threadIdx.x & 63;
        float4 *part = reinterpret_cast<float4 *>(lds) + (threadIdx.x >> 6) * (32 * kCols / 4);
        const uint32_t j = (c0 + wc0) / 2 + lane % kLanes * 8, n = j < half ? min(half - j, 8u) : 0;
        float bx[8] = {}, by[8] = {};
        add_bias(j, bx, by);
#pragma unroll 1
        for (int b = 0; b < TR; ++b) {
            const uint32_t top = r0 + wr0 + 32 * b;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            block_to_lds<TR, TC>(acc, b, part);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (n == 0) continue;
#pragma unroll 1
            for (uint32_t row = lane / kLanes; row < 32; row += kStep) {
                if (top + row >= rows) break;
                float v[16], x[8], y[8];
#pragma unroll
                for (uint32_t q = 0; q < 4; ++q) {
                    const float4 f = part[row * (kCols / 4) + ((lane % kLanes * 4 + q) ^ (row & kMask))];
                    v[4 * q] = f.x, v[4 * q + 1] = f.y, v[4 * q + 2] = f.z, v[4 * q + 3] = f.w;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[i] = v[i] + bx[i];
                    y[i] = v[8 + i] + by[i];
                }
                put(top + row, j, n, x, y);
            }
        }
    }
};
template <class T, bool EXP>
constexpr bool kPaired<GatedEpilogue<T, EXP>> = true;

// The join of a product whose K was cut, as join_kernel's: GROUPS threads a row's sixteen columns.
template <int GROUPS, class Epi>
__global__ __launch_bounds__(kBlock) void join_pairs_kernel(ProductArgs g, Epi epi) {
    constexpr uint32_t kItems = kBlock / GROUPS;
    const uint32_t units = g.ldp / 16, group = threadIdx.x / kItems, e = blockIdx.x * kItems + threadIdx.x % kItems;
    const bool in = e < g.rows * units;
    const uint32_t r = e / units, c = (e - r * units) * 16;
    double s[16] = {};
    if (in) {
        const float *from = g.partial + (uint64_t)r * g.ldp + c;
#pragma unroll 2
        for (uint32_t p = group; p < g.splits; p += GROUPS) {
            const float4 *at = reinterpret_cast<const float4 *>(from + (uint64_t)p * g.rows * g.ldp);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float4 f = at[q];
                s[4 * q] += (double)f.x, s[4 * q + 1] += (double)f.y, s[4 * q + 2] += (double)f.z, s[4 * q + 3] += (double)f.w;
            }
        }
    }
    if constexpr (GROUPS > 1) {
        __shared__ double sums[GROUPS][16][kItems];
#pragma unroll
        for (int i = 0; i < 16; ++i) sums[group][i][threadIdx.x % kItems] = s[i];
        __syncthreads();
        if (group != 0) return;
#pragma unroll
        for (int p = 1; p < GROUPS; ++p)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] += sums[p][i][threadIdx.x];
    }
    if (!in || c / 2 >= epi.half) return;
    float x[8], y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = (float)s[i];
        y[i] = (float)s[8 + i];
    }
    epi.add_bias(c / 2, x, y);
    epi.put(r, c / 2, min(epi.half - c / 2, 8u), x, y);
}

// fp32: output from the projections, a thread four units.
template <bool EXP>
__global__ __launch_bounds__(kBlock) void gate_kernel(const float *sums, float *output, uint32_t rows, uint32_t half, uint32_t fours, Gate gate) {
    for (uint64_t i = (uint64_t)blockIdx.x * kBlock + threadIdx.x; i < (uint64_t)rows * fours; i += (uint64_t)gridDim.x * kBlock) {
        const uint32_t r = (uint32_t)(i / fours), j = (uint32_t)(i - (uint64_t)r * fours) * 4, n = min(half - j, 4u);
        const uint64_t at = (uint64_t)r * 2 * half + j, to = (uint64_t)r * half + j;
        if (n == 4) {
            const f32x4u x = *reinterpret_cast<const f32x4u *>(sums + at), y = *reinterpret_cast<const f32x4u *>(sums + at + half);
            f32x4u z;
#pragma unroll
            for (int e = 0; e < 4; ++e) z[e] = activate_gate<float, EXP>(gate, x[e]) * y[e];
            *reinterpret_cast<f32x4u *>(output + to) = z;
        } else {
            for (uint32_t e = 0; e < n; ++e) output[to + e] = activate_gate<float, EXP>(gate, sums[at + e]) * sums[at + half + e];
        }
    }
}

// fp32, where K is cut: the join of both projections' pieces (in f64) and the output at once, a thread W units of a row or
// GROUPS threads, each taking every GROUPSth piece, for many pieces.
template <int W, int GROUPS, bool EXP>
__global__ __launch_bounds__(kBlock) void gate_join_kernel(const float *partial, uint32_t splits, uint32_t rows, uint32_t half, uint32_t units,
                                                          const float *biases, float *sums, float *output, Gate gate) {
    constexpr uint32_t kAhead = 8 / W, kItems = kBlock / GROUPS;
    const uint32_t i = blockIdx.x * kItems + threadIdx.x % kItems, group = threadIdx.x / kItems, r = i / units, j = (i - r * units) * W;
    const bool in = r < rows;
    const uint64_t at = (uint64_t)r * 2 * half + j, size = (uint64_t)rows * 2 * half;
    double s[2][W] = {};
    for (uint32_t p = group; in && p < splits; p += kAhead * GROUPS) {
        Raw<float, W> x[kAhead][2];  // past the last piece: that one again, not added
#pragma unroll
        for (uint32_t u = 0; u < kAhead; ++u)
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h)
                x[u][h] = *reinterpret_cast<const Raw<float, W> *>(partial + min(p + u * GROUPS, splits - 1) * size + at + h * half);
#pragma unroll
        for (uint32_t u = 0; u < kAhead; ++u)
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
                for (int w = 0; w < W; ++w) s[h][w] += p + u * GROUPS < splits ? (double)x[u][h][w] : 0.0;
    }
    if constexpr (GROUPS > 1) {
        __shared__ double pieces[2][W][kBlock];
#pragma unroll
        for (int w = 0; w < W; ++w) {
            pieces[0][w][threadIdx.x] = s[0][w];
            pieces[1][w][threadIdx.x] = s[1][w];
        }
        __syncthreads();
        if (group != 0) return;
#pragma unroll
        for (uint32_t u = 1; u < GROUPS; ++u)
#pragma unroll
            for (int w = 0; w < W; ++w) {
                s[0][w] += pieces[0][w][threadIdx.x + u * kItems];
                s[1][w] += pieces[1][w][threadIdx.x + u * kItems];
            }
    }
    if (!in) return;
    Raw<float, W> x, y, out;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const float g = (float)s[0][w], u = (float)s[1][w];
        x[w] = biases != nullptr ? g + biases[j + w] : g;
        y[w] = biases != nullptr ? u + biases[half + j + w] : u;
        out[w] = activate_gate<float, EXP>(gate, x[w]) * y[w];
    }
    if (sums != nullptr) {
        *reinterpret_cast<Raw<float, W> *>(sums + at) = x;
        *reinterpret_cast<Raw<float, W> *>(sums + at + half) = y;
    }
    *reinterpret_cast<Raw<float, W> *>(output + (uint64_t)r * half + j) = out;
}

inline uint64_t paired_columns(uint64_t half) { return 2 * round_up(half, 8); }
// Rows of both halves within the loads' 32-bit offsets of a tile's first.
inline bool pairs_direct(const Matrix &x, const Matrix &w, uint64_t half) {
    return operands_direct(x.p, x.ld, w.p, w.ld) && (half + 128) * w.ld < 1u << 30;
}

uint64_t forward_bytes(int type, uint64_t rows, uint64_t inputs, uint64_t hidden) {
    if (type == DKZ_F32) return padded(4 * rows * 2 * hidden) + f32_partial_bytes(rows, 2 * hidden, inputs);
    const uint64_t packed = few_rows(rows) ? 0 : packed_bytes(rows, inputs) + packed_bytes(2 * hidden, inputs);
    return packed + most_partial_bytes(rows, paired_columns(hidden), inputs, true);
}

template <bool EXP>
int forward_f32(hipStream_t stream, uint64_t rows, uint64_t inputs, uint64_t hidden, const Gate &gate, const float *input, const float *weights,
                const float *biases, float *sums, float *output, Workspace ws) {
    constexpr const char *kName = "gated_forward", *kProduct = "gated_forward_product";
    float *own = ws.take<float>(rows * 2 * hidden), *partial = ws.take<float>(f32_partial_bytes(rows, 2 * hidden, inputs) / 4);
    const uint32_t m = (uint32_t)rows, half = (uint32_t)hidden;
    const Tiling t = plan_f32(rows, 2 * hidden, inputs);
    SplitArgs g;
    if (t.splits > 1) {
        DKZ_TRY((run_f32_tiles<kRowMajor, kRowMajor>(stream, kProduct, input, inputs, weights, inputs, 0.0f, (float *)nullptr, 2 * hidden, rows, 2 * hidden,
                                                     inputs, partial, t, g)));
        const auto join = [&](auto kernel, uint32_t width, uint32_t groups) {
            const uint32_t units = half / width;
            return launch_on(stream, kName, kernel, dim3(div_up((uint64_t)m * units, kBlock / groups)), dim3(kBlock), partial, t.splits, m, half, units,
                             biases, sums, output, gate);
        };
        if (t.splits > 32) return join(gate_join_kernel<1, 16, EXP>, 1, 16);
        const bool fours = hidden % 4 == 0 && aligned16(output) && aligned16(sums);
        return fours ? join(gate_join_kernel<4, 1, EXP>, 4, 1) : join(gate_join_kernel<1, 1, EXP>, 1, 1);
    }
    if (sums == nullptr) sums = own;
    LinearEpilogue<float, false> e;
    e.biases = biases;
    e.residual = nullptr;
    e.activated = nullptr;
    e.output = sums;
    e.ld = 2 * half;
    e.act = kLinear;
    e.words = true;
    e.draws = make_draws(0.0f, 1.0f, 0, 0);
    DKZ_TRY((run_f32_tiles<kRowMajor, kRowMajor>(stream, kProduct, input, inputs, weights, inputs, 0.0f, (float *)nullptr, 2 * hidden, rows, 2 * hidden,
                                                 inputs, partial, t, g, e)));
    if (t.stream) DKZ_TRY(join_f32_stream(stream, kProduct, t, g, e));
    const uint64_t fours = (hidden + 3) / 4;
    const dim3 grid((uint32_t)std::min<uint64_t>((rows * fours + kBlock - 1) / kBlock, 1u << 16));
    return launch_on(stream, kName, gate_kernel<EXP>, grid, dim3(kBlock), sums, output, m, half, (uint32_t)fours, gate);
}

template <bool EXP>
int forward_bf16(hipStream_t stream, uint64_t rows, uint64_t inputs, uint64_t hidden, const Gate &gate, const __bf16 *input, const __bf16 *weights,
                 const float *biases, __bf16 *sums, __bf16 *output, Workspace ws) {
    constexpr const char *kName = "gated_forward";
    typedef GatedEpilogue<__bf16, EXP> Epi;
    Matrix x{input, inputs}, w{weights, inputs};
    if (!few_rows(rows)) DKZ_TRY(pack(stream, x, rows, w, 2 * hidden, inputs, ws));
    const uint64_t cols = paired_columns(hidden);
    const ProductPlan p = plan_product(rows, cols, inputs, true, true, pairs_direct(x, w, hidden));
    float *partial = ws.take<float>(p.partial_bytes(rows, cols) / 4);
    const Epi epi{biases, sums, output, (uint32_t)hidden, gate};
    const Product product{x.p, x.ld, w.p, w.ld, rows, cols, inputs};
    DKZ_TRY((run_product<false, false>(stream, kName, product, p, partial, epi)));
    if (p.splits <= 1 || p.skinny()) return 0;
    const ProductArgs g = product_args(product, p, partial);
    const uint64_t units = rows * (g.ldp / 16);
    if (p.splits > 4) return launch_on(stream, kName, join_pairs_kernel<8, Epi>, dim3(div_up(units, kBlock / 8)), dim3(kBlock), g, epi);
    return launch_on(stream, kName, join_pairs_kernel<1, Epi>, dim3(div_up(units, kBlock)), dim3(kBlock), g, epi);
}

// ---- backward ----

constexpr uint32_t kDeltaRows = 64;    // rows a workgroup of gate_delta_kernel takes at once,
constexpr uint32_t kDeltaFew = 16;     // or, where that makes few workgroups
constexpr uint32_t kDeltaWhole = 128;  // rows up to which it takes all of its units'
constexpr uint32_t kDeltaFill = 128;   // workgroups that are enough for eight units a thread

template <class T>
struct GateDelta {
    const T *sums, *delta;
    uint32_t rows, half;
    Gate gate;
    T *d;  // null: not wanted
    uint32_t ldd, blocks_c, blocks;
    float beta, *to;  // null: not wanted
    PackArgs pack;    // of T bf16: copies that the products need too, by the workgroups after the first `blocks`
};

// d(r, j) and d(r, half + j) to d, in rows of ldd (ldd's padding is 0), and the sums of ROWS rows' columns to `to`. bf16: d is
// rounded as it is stored, since the matrix instruction takes no wider operands (two of them a d would double the products'
// time): the gradients are off by 0.0023 of their norm, by their own rounding alone 0.0017. The sums take it unrounded. A
// thread takes W units of eight rows; the eight sums of a unit's threads are added in row order. WHOLE: a workgroup takes all rows,
// adds their sums in f64, and `to` is bias_updates itself. Bound by memory where it is large: 4096 rows of 8192 units, bf16, 56 us
// (6.0 TB/s).
template <class T, int W, bool EXP, bool WHOLE, uint32_t ROWS>
__global__ __launch_bounds__(kBlock) void gate_delta_kernel(GateDelta<T> g) {
    constexpr uint32_t kLanes = 32, kGroups = kBlock / kLanes, kEach = ROWS / kGroups;
    __shared__ float lds[2][kGroups][kLanes * W + 4];
    if constexpr (sizeof(T) == 2) {
        if (blockIdx.x >= g.blocks) return pack_chunk(g.pack, (blockIdx.x - g.blocks) * kBlock + threadIdx.x);
    }
    const uint32_t half = g.half, x = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
    const uint32_t block_r = blockIdx.x / g.blocks_c, block_c = blockIdx.x - block_r * g.blocks_c;
    const uint32_t j = (block_c * kLanes + x) * W;
    const bool in = j < half;  // W == 8: half is a multiple of it
    constexpr uint32_t kBatch = W == 1 ? kEach : 2;  // rows whose loads are on their way at once
    constexpr uint32_t kStored = (2 * kLanes * W + kBlock - 1) / kBlock;  // sums that a thread stores
    double whole[kStored] = {};
    for (uint32_t top = WHOLE ? 0 : block_r * ROWS; top < g.rows; top += ROWS) {
        const uint32_t r0 = top + group * kEach;
        float total[2][W] = {};
#pragma unroll 1
        for (uint32_t i0 = 0; i0 < kEach; i0 += kBatch) {
            Raw<T, W> s[kBatch], up[kBatch], dl[kBatch];
#pragma unroll
            for (uint32_t i = 0; i < kBatch; ++i) {
                const uint64_t r = min(r0 + i0 + i, g.rows - 1), at = in ? j : 0;
                load_raw<T, RowRun, W>(g.sums, RowRun{r * 2 * half + at, W}, s[i]);
                load_raw<T, RowRun, W>(g.sums, RowRun{r * 2 * half + half + at, W}, up[i]);
                load_raw<T, RowRun, W>(g.delta, RowRun{r * half + at, W}, dl[i]);
            }
#pragma unroll
            for (uint32_t i = 0; i < kBatch; ++i) {
                const uint32_t r = r0 + i0 + i;
                if (r >= g.rows || !in) break;
                float dg[W], du[W];
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    float a;
                    const float slope = gate_slope<T, EXP>(g.gate, (float)s[i][w], a), v = (float)dl[i][w];
                    dg[w] = v * (float)up[i][w] * slope;
                    du[w] = v * a;
                    total[0][w] += dg[w];
                    total[1][w] += du[w];
                }
                if (g.d != nullptr) {
                    store_n(g.d, RowRun{(uint64_t)r * g.ldd + j, W}, dg);
                    store_n(g.d, RowRun{(uint64_t)r * g.ldd + half + j, W}, du);
                }
            }
        }
        // The padding, at most seven elements a row.
        if (g.d != nullptr && block_c == 0 && 2 * half + x < g.ldd)
            for (uint32_t i = 0; i < kEach; ++i)
                if (r0 + i < g.rows) store1(g.d, (uint64_t)(r0 + i) * g.ldd + 2 * half + x, 0.0f);
        if (g.to != nullptr) {
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int w = 0; w < W; ++w) lds[s][group][x * W + w] = total[s][w];
            __syncthreads();
#pragma unroll
            for (uint32_t i = 0; i < kStored; ++i) {
                const uint32_t e = threadIdx.x + i * kBlock, s = e / (kLanes * W), c = e % (kLanes * W), unit = block_c * kLanes * W + c;
                if (s >= 2 || unit >= half) continue;
                float t = lds[s][0][c];
#pragma unroll
                for (uint32_t k = 1; k < kGroups; ++k) t += lds[s][k][c];
                if constexpr (WHOLE) whole[i] += (double)t;
                else g.to[(uint64_t)block_r * 2 * half + s * half + unit] = t;
            }
            if constexpr (WHOLE) __syncthreads();
        }
        if constexpr (!WHOLE) break;
    }
    if constexpr (WHOLE) {
        if (g.to == nullptr) return;
#pragma unroll
        for (uint32_t i = 0; i < kStored; ++i) {
            const uint32_t e = threadIdx.x + i * kBlock, s = e / (kLanes * W), unit = block_c * kLanes * W + e % (kLanes * W);
            if (s >= 2 || unit >= half) continue;
            float &to = g.to[s * half + unit];
            to = g.beta == 0.0f ? (float)whole[i] : g.beta * to + (float)whole[i];
        }
    }
}

// Rows a workgroup takes, eight units a thread: 64 where that fills the chip; 16 else, whose loads wait in parallel and not one
// after another (512 rows of 4096 units 10.0 -> 7.3 us). Not for single units, whose 64 rows' loads are on their way at once
// (333 rows of 1503 8.6 -> 8.4, and more sums to add: 28.1 -> 28.6 with the products).
inline uint32_t delta_rows(uint64_t rows, uint64_t half) {
    const uint64_t blocks_c = div_up(half, 256);
    const bool few = rows > kDeltaWhole && half % 8 == 0 && div_up(rows, kDeltaRows) * blocks_c < 512 && div_up(rows, kDeltaFew) * blocks_c >= kDeltaFill;
    return few ? kDeltaFew : kDeltaRows;
}
inline uint64_t delta_ld(int type, uint64_t hidden) { return round_up(2 * hidden, type == DKZ_F32 ? 4 : 8); }

struct BackwardPlan {
    uint64_t d_bytes, sum_bytes, packed, partial_bytes;
    uint64_t total() const { return d_bytes + sum_bytes + packed + partial_bytes; }
};
BackwardPlan backward_plan(int type, uint64_t rows, uint64_t inputs, uint64_t hidden) {
    BackwardPlan p;
    const uint64_t n = 2 * hidden;
    p.d_bytes = padded(rows * delta_ld(type, hidden) * type_size(type));
    p.sum_bytes = padded(4 * n * div_up(rows, delta_rows(rows, hidden)));
    p.packed = type == DKZ_F32 || rows == 0 ? 0 : packed_bytes(rows, inputs) + packed_bytes(n, inputs);
    if (type == DKZ_F32)
        p.partial_bytes = std::max(f32_partial_bytes(rows, inputs, n), f32_partial_bytes(n, inputs, rows));
    else
        p.partial_bytes = std::max(most_partial_bytes(rows, inputs, n, false), most_partial_bytes(n, inputs, rows, false));
    return p;
}

// Sums of rows' columns that are still to be added up, to bias_updates (as column_sums); cols 0: none.
struct BiasSums {
    const float *partial;
    uint32_t chunks, cols;
    float beta, *to;
};

// bias_updates null: not wanted; sums: room for the sums of every delta_rows rows, `left` what is to be done with them.
template <class T, bool EXP>
int run_gate_delta(hipStream_t stream, GateDelta<T> g, float *sums, float *bias_updates, BiasSums &left) {
    constexpr const char *kName = "gated_backward_delta";
    const bool whole = g.rows <= kDeltaWhole;
    const uint32_t each = delta_rows(g.rows, g.half), blocks_r = whole ? 1 : div_up(g.rows, each);
    const bool eights = g.half % 8 == 0 && (each == kDeltaFew || div_up(g.half, 256) * blocks_r >= kDeltaFill);
    g.blocks_c = div_up(g.half, eights ? 256 : 32);
    g.blocks = g.blocks_c * blocks_r;
    g.to = bias_updates == nullptr ? nullptr : whole ? bias_updates : sums;
    const dim3 grid(g.blocks + div_up(g.pack.count(), kBlock)), block(kBlock);
    const auto run = [&](auto kernel) { return launch_on(stream, kName, kernel, grid, block, g); };
    if (whole) return eights ? run(gate_delta_kernel<T, 8, EXP, true, kDeltaRows>) : run(gate_delta_kernel<T, 1, EXP, true, kDeltaRows>);
    DKZ_TRY(each == kDeltaFew ? run(gate_delta_kernel<T, 8, EXP, false, kDeltaFew>)
            : eights          ? run(gate_delta_kernel<T, 8, EXP, false, kDeltaRows>)
                              : run(gate_delta_kernel<T, 1, EXP, false, kDeltaRows>));
    if (bias_updates != nullptr) left = {sums, blocks_r, 2 * g.half, g.beta, bias_updates};
    return 0;
}

// Both gradients, as product_pair_kernel, and, by the workgroups after their `groups`, the bias sums that are left (333x1001, 1503 units 28.1 -> 26.0 us
// without a launch of theirs).
template <class T, class Epi>
__global__ __launch_bounds__(T::kThreads, 2) void gradients_kernel(ProductArgs a, Epi epi_a, ProductArgs b, Epi epi_b, uint32_t tiles_a, bool a_first,
                                                                  uint32_t groups, BiasSums s) {
    static_assert(T::kThreads == kBlock && lds_bytes<T, true>() >= sizeof(double[kSumGroups][kSumLanes]));
    __shared__ __align__(1024) char lds[lds_bytes<T, true>()];
    if (blockIdx.x >= groups)
        return column_sums(s.partial, s.chunks, s.cols, s.beta, s.to, blockIdx.x - groups, *reinterpret_cast<double(*)[kSumGroups][kSumLanes]>(lds));
    const uint32_t first = a_first ? tiles_a : groups - tiles_a, block = blockIdx.x < first ? blockIdx.x : blockIdx.x - first;
    if ((blockIdx.x < first) == a_first) product_tile<T, false, true, true>(a, epi_a, block, lds);
    else product_tile<T, true, true, true>(b, epi_b, block, lds);
}
struct GradientsLaunch {
    BiasSums &left;
    template <class T, class Epi>
    int run(hipStream_t stream, const char *name, const ProductArgs &a, const Epi &epi_a, const ProductArgs &b, const Epi &epi_b, uint32_t groups_a,
            uint32_t groups_b, bool a_first) {
        const BiasSums s = left;
        left = {};
        const uint32_t groups = groups_a + groups_b;
        return launch_on(stream, name, gradients_kernel<T, Epi>, dim3(groups + div_up(s.cols, kSumLanes)), dim3(kBlock), a, epi_a, b, epi_b, groups_a,
                         a_first, groups, s);
    }
};

template <class T>
int backward(hipStream_t stream, int type, uint64_t rows, uint64_t inputs, uint64_t hidden, int act, const void *input, const void *weights,
             const void *sums_in, const void *delta_in, const void *input_residual, float beta, float *bias_updates, void *weight_updates,
             void *input_delta, Workspace ws) {
    const BackwardPlan plan = backward_plan(type, rows, inputs, hidden);
    T *d = ws.take<T>(plan.d_bytes / sizeof(T));
    float *sums = ws.take<float>(plan.sum_bytes / 4), *partial = ws.take<float>(plan.partial_bytes / 4);
    const uint64_t ldd = delta_ld(type, hidden), n = 2 * hidden;
    const bool products = inputs != 0 && (weight_updates != nullptr || input_delta != nullptr);
    Matrix x{weight_updates != nullptr ? reinterpret_cast<const __bf16 *>(input) : nullptr, inputs};
    Matrix w{input_delta != nullptr ? reinterpret_cast<const __bf16 *>(weights) : nullptr, inputs};
    BiasSums left{};
    if (rows != 0 && hidden != 0 && (products || bias_updates != nullptr)) {
        GateDelta<T> g{};
        g.sums = static_cast<const T *>(sums_in);
        g.delta = static_cast<const T *>(delta_in);
        g.rows = (uint32_t)rows;
        g.half = (uint32_t)hidden;
        g.gate = make_gate(act);
        g.d = products ? d : nullptr;
        g.ldd = (uint32_t)ldd;
        g.beta = beta;
        if (sizeof(T) == 2 && products) g.pack = pack_args(x, rows, w, n, inputs, ws);
        DKZ_TRY(gate_has_exp(act) ? (run_gate_delta<T, true>(stream, g, sums, bias_updates, left)) : (run_gate_delta<T, false>(stream, g, sums, bias_updates, left)));
    } else if (bias_updates != nullptr) {
        DKZ_TRY(add_column_sums(stream, sums, 0, n, beta, bias_updates));  // no rows: beta * bias_updates
    }
    constexpr const char *kWeights = "gated_backward_weights", *kInput = "gated_backward_input";
    if constexpr (sizeof(T) == 4) {
        const T *in = static_cast<const T *>(input), *wt = static_cast<const T *>(weights);
        if (weight_updates != nullptr)
            DKZ_TRY((run_f32<kColMajor, kColMajor>(stream, kWeights, d, ldd, in, inputs, beta, static_cast<float *>(weight_updates), inputs, n, inputs,
                                                   rows, partial)));
        if (input_delta != nullptr)
            DKZ_TRY((run_f32<kRowMajor, kColMajor>(stream, kInput, d, ldd, wt, inputs, 0.0f, (float *)nullptr, inputs, rows, inputs, n, partial,
                                                   store_epilogue<T>(input_delta, input_residual, inputs, 0.0f))));
    } else {
        const Product to_input{d, ldd, w.p, w.ld, rows, inputs, n}, to_weights{d, ldd, x.p, x.ld, n, inputs, rows};
        DKZ_TRY(run_gradients(stream, kInput, input_delta != nullptr ? &to_input : nullptr, store_epilogue<T>(input_delta, input_residual, inputs, 0.0f),
                              kWeights, weight_updates != nullptr ? &to_weights : nullptr, store_epilogue<T>(weight_updates, nullptr, inputs, beta), partial, true, GradientsLaunch{left}));
    }
    return left.cols != 0 ? add_column_sums(stream, left.partial, left.chunks, left.cols, left.beta, left.to) : 0;
}

bool sizes_ok(int type, int rows, int inputs, int hidden) {
    if (!type_ok(type) || rows < 0 || inputs < 0 || hidden < 0 || rows > 1 << 26 || inputs > 1 << 26 || hidden > 1 << 25) return false;
    const uint64_t m = (uint64_t)rows, k = (uint64_t)inputs, n = 2 * (uint64_t)hidden;
    return m * k + 3 <= kMaxElems && n * k + 3 <= kMaxElems && m * n + 3 <= kMaxElems;
}

}  // namespace
}  // namespace dkz

using namespace dkz;

extern "C" {

int dkz_gated_forward_workspace(int type, int rows, int inputs, int hidden, size_t *bytes) {
    DKZ_REQUIRE(bytes != nullptr && sizes_ok(type, rows, inputs, hidden));
    *bytes = (size_t)forward_bytes(type, (uint64_t)rows, (uint64_t)inputs, (uint64_t)hidden);
    return 0;
}

int dkz_gated_forward(int type, int rows, int inputs, int hidden, int activation, const void *input, const void *weights,
                      const float *biases, void *sums, void *output, void *workspace, size_t workspace_bytes) {
    DKZ_REQUIRE(sizes_ok(type, rows, inputs, hidden));
    DKZ_REQUIRE(gate_ok(activation));
    if (rows == 0 || hidden == 0) return 0;
    DKZ_REQUIRE(output != nullptr && (inputs == 0 || (input != nullptr && weights != nullptr)));
    const uint64_t m = (uint64_t)rows, k = (uint64_t)inputs, n = (uint64_t)hidden, size = type_size(type), need = forward_bytes(type, m, k, n);
    DKZ_REQUIRE_WORKSPACE(need);
    const Span writes[] = {{output, m * n * size}, {sums, 2 * m * n * size}, {workspace, need}};
    const Span reads[] = {{input, m * k * size}, {weights, 2 * n * k * size}, {biases, 8 * n}};
    DKZ_REQUIRE(disjoint(writes, reads));
    const Workspace ws{static_cast<char *>(workspace), need};
    const Gate gate = make_gate(activation);
    const hipStream_t stream = current_stream();
    const auto run = [&](auto exp) {
        constexpr bool kExp = decltype(exp)::value;
        if (type == DKZ_F32)
            return forward_f32<kExp>(stream, m, k, n, gate, static_cast<const float *>(input), static_cast<const float *>(weights), biases,
                                     static_cast<float *>(sums), static_cast<float *>(output), ws);
        return forward_bf16<kExp>(stream, m, k, n, gate, static_cast<const __bf16 *>(input), static_cast<const __bf16 *>(weights), biases,
                                  static_cast<__bf16 *>(sums), static_cast<__bf16 *>(output), ws);
    };
    return gate_has_exp(activation) ? run(std::true_type{}) : run(std::false_type{});
}

int dkz_gated_backward_workspace(int type, int rows, int inputs, int hidden, size_t *bytes) {
    DKZ_REQUIRE(bytes != nullptr && sizes_ok(type, rows, inputs, hidden));
    *bytes = (size_t)backward_plan(type, (uint64_t)rows, (uint64_t)inputs, (uint64_t)hidden).total();
    return 0;
}

int dkz_gated_backward(int type, int rows, int inputs, int hidden, int activation, const void *input, const void *weights,
                       const void *sums, const void *delta, const void *input_residual, float beta, float *bias_updates,
                       void *weight_updates, void *input_delta, void *workspace, size_t workspace_bytes) {
    DKZ_REQUIRE(sizes_ok(type, rows, inputs, hidden));
    DKZ_REQUIRE(gate_ok(activation));
    const uint64_t m = (uint64_t)rows, k = (uint64_t)inputs, n = (uint64_t)hidden, size = type_size(type);
    const uint64_t in = m * k * size, w = 2 * n * k * size, out = m * n * size;
    const bool products = out != 0 && in + w != 0 && (weight_updates != nullptr || input_delta != nullptr);
    if (out != 0 && (products || bias_updates != nullptr)) {
        DKZ_REQUIRE(delta != nullptr && sums != nullptr);
        DKZ_REQUIRE(in == 0 || weight_updates == nullptr || input != nullptr);
        DKZ_REQUIRE(w == 0 || input_delta == nullptr || weights != nullptr);
    }
    const uint64_t need = backward_plan(type, m, k, n).total();
    DKZ_REQUIRE_WORKSPACE(need);
    const Span writes[] = {{bias_updates, 8 * n}, {weight_updates, w}, {input_delta, in}, {workspace, need}};
    const Span reads[] = {{input, in}, {weights, w}, {sums, 2 * out}, {delta, out}, {input_residual == input_delta ? nullptr : input_residual, in}};
    DKZ_REQUIRE(disjoint(writes, reads));
    const Workspace ws{static_cast<char *>(workspace), need};
    const hipStream_t stream = current_stream();
    if (type == DKZ_F32)
        return backward<float>(stream, type, m, k, n, activation, input, weights, sums, delta, input_residual, beta, bias_updates, weight_updates,
                               input_delta, ws);
    return backward<__bf16>(stream, type, m, k, n, activation, input, weights, sums, delta, input_residual, beta, bias_updates, weight_updates,
                            input_delta, ws);
}

}  // extern "C"
