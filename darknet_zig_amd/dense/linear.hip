// linear.hip -- a connected layer with its epilogue in the product (bias,
// activation, dropout, residual), and its backward pass.
#include <math.h>

#include <utility>

#include "dense_internal.hpp"
#include "epilogue.hpp"
#include "product_plan.hpp"
#include "product_f32.hpp"

namespace dkz {
namespace {

template <class T, bool EXP>
LinearEpilogue<T, EXP> linear_epilogue(uint64_t outputs, int act, const Draws &draws, const float *biases,
                                       const void *residual, void *activated, void *output) {
    LinearEpilogue<T, EXP> e;
    e.biases = biases;
    e.residual = static_cast<const T *>(residual);
    e.activated = static_cast<T *>(activated);
    e.output = static_cast<T *>(output);
    e.ld = (uint32_t)outputs;
    e.act = act;
    e.words = rows_in_words<T>(outputs, residual, activated, output);
    e.draws = draws;
    return e;
}

template <bool EXP>
int forward(hipStream_t stream, int type, uint64_t rows, uint64_t inputs, uint64_t outputs, int act, const Draws &draws, const void *input,
            const void *weights, const float *biases, const void *residual, void *activated, void *output, Workspace ws) {
    constexpr const char *kName = "linear_forward";
    if (type == DKZ_F32) {
        float *partial = ws.take<float>(f32_partial_bytes(rows, outputs, inputs) / 4);
        return run_f32<kRowMajor, kRowMajor>(stream, kName, static_cast<const float *>(input), inputs,
                                             static_cast<const float *>(weights), inputs, 0.0f, (float *)nullptr, outputs, rows,
                                             outputs, inputs, partial,
                                             linear_epilogue<float, EXP>(outputs, act, draws, biases, residual, activated, output));
    }
    Matrix x{static_cast<const __bf16 *>(input), inputs}, w{static_cast<const __bf16 *>(weights), inputs};
    if (!few_rows(rows)) DKZ_TRY(pack(stream, x, rows, w, outputs, inputs, ws));
    const ProductPlan p = plan_product(rows, outputs, inputs, true, true, operands_direct(x.p, x.ld, w.p, w.ld));
    float *partial = ws.take<float>(p.partial_bytes(rows, outputs) / 4);
    return run_product<false, false>(stream, kName, {x.p, x.ld, w.p, w.ld, rows, outputs, inputs}, p, partial,
                                     linear_epilogue<__bf16, EXP>(outputs, act, draws, biases, residual, activated, output));
}

uint64_t forward_bytes(int type, uint64_t rows, uint64_t inputs, uint64_t outputs) {
    if (type == DKZ_F32) return f32_partial_bytes(rows, outputs, inputs);
    const uint64_t packed = few_rows(rows) ? 0 : packed_bytes(rows, inputs) + packed_bytes(outputs, inputs);
    return packed + most_partial_bytes(rows, outputs, inputs, true);
}

// ---- backward ----

constexpr uint32_t kDeltaRows = 64;   // rows a workgroup of delta_kernel takes at once
constexpr uint32_t kDeltaWhole = 128;  // rows up to which it takes all of its columns'
constexpr uint32_t kDeltaFill = 128;   // workgroups that are enough for eight columns a thread

// d = dropout(delta) * gradient(activated), stored to d (null: not) in rows of
// ldd, and sum_scale times the sums of kDeltaRows rows' columns to `to` (null: not). Bound by
// memory: a thread takes W columns of eight rows, all of its loads issued before
// the first is used; the eight sums of a column's threads are added in row order.
// W is eight where rows are whole eights and that leaves workgroups for the chip
// (8192x4096 48 us), else one (250x1024 with leaky and dropout: the backward pass 16
// us, 33 with eight). WHOLE: a workgroup takes all rows, adds their sums in f64 and
// `to` is bias_updates itself: a launch less where there are few rows.
template <class T, int W, bool WHOLE>
__global__ __launch_bounds__(kBlock) void delta_kernel(const T *delta, const T *activated, uint32_t rows, uint32_t cols, int act,
                                                      Draws draws, T *d, uint32_t ldd, uint32_t blocks_c, float sum_scale, float beta,
                                                      float *to) {
    constexpr uint32_t kLanes = 32, kGroups = kBlock / kLanes, kEach = kDeltaRows / kGroups;
    __shared__ float sums[kGroups][kLanes * W + 4];
    const uint32_t x = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
    const uint32_t block_r = blockIdx.x / blocks_c, block_c = blockIdx.x - block_r * blocks_c;
    const uint32_t c = (block_c * kLanes + x) * W;
    const bool in = c < cols;  // W == 8: cols is a multiple of it, and ldd is cols
    const uint32_t column = block_c * kLanes * W + threadIdx.x;  // whose sum this thread stores
    const bool stores = threadIdx.x < kLanes * W && column < cols;
    static_assert(kLanes * W <= kBlock, "a thread a column");
    double total = 0.0;
    for (uint32_t top = WHOLE ? 0 : block_r * kDeltaRows; top < rows; top += kDeltaRows) {
        const uint32_t r0 = top + group * kEach;
        Raw<T, W> v[kEach], y[kEach];
        float s[W] = {};
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            const RowRun e{(uint64_t)min(r0 + i, rows - 1) * cols + (in ? c : 0), W};
            load_raw<T, RowRun, W>(delta, e, v[i]);
            if (act != kLinear) load_raw<T, RowRun, W>(activated, e, y[i]);
        }
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            const uint32_t r = r0 + i;
            if (r >= rows) break;
            float g[W], a[W];
#pragma unroll
            for (int w = 0; w < W; ++w) g[w] = (float)v[i][w];
            draws.run(g, (uint64_t)r * cols + c);
            if (act != kLinear) {
#pragma unroll
                for (int w = 0; w < W; ++w) a[w] = (float)y[i][w];
                gradient_all(act, a, g);
            }
#pragma unroll
            for (int w = 0; w < W; ++w) {
                if (!in) g[w] = 0.0f;  // the rows' padding
                s[w] += g[w];
            }
            if (d != nullptr && c < ldd) store_n(d, RowRun{(uint64_t)r * ldd + c, W}, g);
        }
        if (to != nullptr) {
#pragma unroll
            for (int w = 0; w < W; ++w) sums[group][x * W + w] = s[w];
            __syncthreads();
            if (stores) {
                float t = sums[0][threadIdx.x];
#pragma unroll
                for (uint32_t i = 1; i < kGroups; ++i) t += sums[i][threadIdx.x];
                t *= sum_scale;
                if constexpr (WHOLE) total += (double)t;
                else to[(uint64_t)block_r * cols + column] = t;
            }
            if constexpr (WHOLE) __syncthreads();
        }
        if constexpr (!WHOLE) break;
    }
    if (WHOLE && to != nullptr && stores) to[column] = beta == 0.0f ? (float)total : beta * to[column] + (float)total;
}

// bias_updates null: not wanted; sums: room for the sums of every kDeltaRows rows.
template <class T>
int run_delta(hipStream_t stream, const T *delta, const T *activated, uint64_t rows, uint64_t cols, int act, const Draws &draws,
              T *d, uint64_t ldd, float sum_scale, float *sums, float beta, float *bias_updates) {
    constexpr const char *kName = "linear_backward_delta";
    const bool whole = rows <= kDeltaWhole;
    const uint32_t blocks_r = whole ? 1 : div_up(rows, kDeltaRows);
    const bool eights = cols % 8 == 0 && div_up(cols, 32 * 8) * blocks_r >= kDeltaFill;
    const uint32_t blocks_c = div_up(eights ? cols : ldd, eights ? 32 * 8 : 32);
    const dim3 grid(blocks_c * blocks_r), block(kBlock);
    const auto run = [&](auto kernel) {
        return launch_on(stream, kName, kernel, grid, block, delta, activated, (uint32_t)rows, (uint32_t)cols, act, draws, d, (uint32_t)ldd,
                         blocks_c, sum_scale, beta, bias_updates == nullptr ? nullptr : whole ? bias_updates : sums);
    };
    if (whole) return eights ? run(delta_kernel<T, 8, true>) : run(delta_kernel<T, 1, true>);
    DKZ_TRY(eights ? run(delta_kernel<T, 8, false>) : run(delta_kernel<T, 1, false>));
    return bias_updates != nullptr ? add_column_sums(stream, sums, div_up(rows, kDeltaRows), cols, beta, bias_updates) : 0;
}

// Leading dimension of d in the workspace: whole 16-byte chunks.
inline uint64_t delta_ld(int type, uint64_t outputs) { return round_up(outputs, type == DKZ_F32 ? 4 : 8); }

struct BackwardPlan {
    uint64_t d_bytes, sum_bytes, packed, partial_bytes;
    uint64_t total() const { return d_bytes + sum_bytes + packed + partial_bytes; }
};
BackwardPlan backward_plan(int type, uint64_t rows, uint64_t inputs, uint64_t outputs) {
    BackwardPlan p;
    p.d_bytes = padded(rows * delta_ld(type, outputs) * type_size(type));
    p.sum_bytes = padded(4 * outputs * div_up(rows, kDeltaRows));
    p.packed = type == DKZ_F32 || rows == 0 ? 0 : packed_bytes(rows, inputs) + packed_bytes(outputs, inputs);
    if (type == DKZ_F32)
        p.partial_bytes = std::max(f32_partial_bytes(rows, inputs, outputs), f32_partial_bytes(outputs, inputs, rows));
    else
        p.partial_bytes = std::max(most_partial_bytes(rows, inputs, outputs, false), most_partial_bytes(outputs, inputs, rows, false));
    return p;
}

template <class T>
int backward(hipStream_t stream, int type, uint64_t rows, uint64_t inputs, uint64_t outputs, int act, const Draws &draws, const void *input,
             const void *weights, const void *activated, const void *delta, const void *input_residual, float beta,
             float *bias_updates, void *weight_updates, void *input_delta, Workspace ws) {
    const BackwardPlan plan = backward_plan(type, rows, inputs, outputs);
    T *d = ws.take<T>(plan.d_bytes / sizeof(T));
    float *sums = ws.take<float>(plan.sum_bytes / 4), *partial = ws.take<float>(plan.partial_bytes / 4);
    uint64_t ldd = delta_ld(type, outputs);
    const bool products = inputs != 0 && (weight_updates != nullptr || input_delta != nullptr);
    // bf16 products take d / scale, and their results are multiplied by the scale in fp32: where the gradient is 0 or 1 (linear, relu)
    // d / scale is a delta or 0 and needs no rounding, and an input or weight gradient is off by its own rounding alone (8192x4096x4096
    // with dropout, distance from 64 bits: 0.0024 with d rounded, 0.0017 so). Other gradients' d is rounded to bf16, as any operand of
    // a bf16 product has to be. A scale far from 1 stays with d: a sum that it keeps below fp32's largest value, or above its smallest,
    // would not be there without it, and an infinite one (all dropped) times sums of 0 is no 0.
    Draws inner = draws;
    float alpha = 1.0f;
    if (sizeof(T) == 2 && fabsf(draws.scale) >= 0x1p-8f && fabsf(draws.scale) <= 0x1p8f) std::swap(alpha, inner.scale);
    // The delta itself where nothing changes it and its rows lie on 16-byte boundaries.
    const bool same = act == kLinear && inner.limit == 0 && inner.scale == 1.0f && ldd == outputs && aligned16(delta);
    if (same || !products) {
        d = nullptr;
        ldd = outputs;
    }
    if (rows != 0 && outputs != 0 && (bias_updates != nullptr || d != nullptr))
        DKZ_TRY(run_delta(stream, static_cast<const T *>(delta), static_cast<const T *>(activated), rows, outputs, act, inner, d, ldd,
                          alpha, sums, beta, bias_updates));
    else if (bias_updates != nullptr)
        DKZ_TRY(add_column_sums(stream, sums, 0, outputs, beta, bias_updates));  // no rows: beta * bias_updates
    const T *dd = d != nullptr ? d : static_cast<const T *>(delta);
    constexpr const char *kWeights = "linear_backward_weights", *kInput = "linear_backward_input";
    if constexpr (sizeof(T) == 4) {
        const T *x = static_cast<const T *>(input), *w = static_cast<const T *>(weights);
        if (weight_updates != nullptr)
            DKZ_TRY((run_f32<kColMajor, kColMajor>(stream, kWeights, dd, ldd, x, inputs, beta, static_cast<float *>(weight_updates),
                                                   inputs, outputs, inputs, rows, partial)));
        if (input_delta != nullptr)
            DKZ_TRY((run_f32<kRowMajor, kColMajor>(stream, kInput, dd, ldd, w, inputs, 0.0f, (float *)nullptr, inputs, rows, inputs,
                                                   outputs, partial, store_epilogue<T>(input_delta, input_residual, inputs, 0.0f))));
    } else {
        Matrix x{weight_updates != nullptr ? static_cast<const T *>(input) : nullptr, inputs};
        Matrix w{input_delta != nullptr ? static_cast<const T *>(weights) : nullptr, inputs};
        if (rows != 0) DKZ_TRY(pack(stream, x, rows, w, outputs, inputs, ws));
        const Product to_input{dd, ldd, w.p, w.ld, rows, inputs, outputs}, to_weights{dd, ldd, x.p, x.ld, outputs, inputs, rows};
        const auto epi_input = store_epilogue<T>(input_delta, input_residual, inputs, 0.0f, alpha);
        const auto epi_weights = store_epilogue<T>(weight_updates, nullptr, inputs, beta, alpha);
        DKZ_TRY(run_gradients(stream, kInput, input_delta != nullptr ? &to_input : nullptr, epi_input, kWeights,
                              weight_updates != nullptr ? &to_weights : nullptr, epi_weights, partial));
    }
    return 0;
}

}  // namespace
}  // namespace dkz

using namespace dkz;

extern "C" {

int dkz_linear_forward_workspace(int type, int rows, int inputs, int outputs, size_t *bytes) {
    DKZ_REQUIRE(bytes != nullptr && type_ok(type) && rows >= 0 && inputs >= 0 && outputs >= 0);
    DKZ_REQUIRE_SIDE(rows);
    DKZ_REQUIRE_SIDE(inputs);
    DKZ_REQUIRE_SIDE(outputs);
    DKZ_REQUIRE_ELEMS(rows, inputs);
    DKZ_REQUIRE_ELEMS(outputs, inputs);
    DKZ_REQUIRE_ELEMS(rows, outputs);
    *bytes = (size_t)forward_bytes(type, (uint64_t)rows, (uint64_t)inputs, (uint64_t)outputs);
    return 0;
}

int dkz_linear_forward(int type, int rows, int inputs, int outputs, int activation, float prob, float scale, unsigned int seed,
                       unsigned long long first, const void *input, const void *weights, const float *biases,
                       const void *residual, void *activated, void *output, void *workspace, size_t workspace_bytes) {
    DKZ_REQUIRE(type_ok(type) && rows >= 0 && inputs >= 0 && outputs >= 0);
    DKZ_REQUIRE(activation >= 0 && activation < kActCount);
    DKZ_REQUIRE_SIDE(rows);
    DKZ_REQUIRE_SIDE(inputs);
    DKZ_REQUIRE_SIDE(outputs);
    DKZ_REQUIRE_ELEMS(rows, inputs);
    DKZ_REQUIRE_ELEMS(outputs, inputs);
    DKZ_REQUIRE_ELEMS(rows, outputs);
    if (rows == 0 || outputs == 0) return 0;
    DKZ_REQUIRE(output != nullptr && (inputs == 0 || (input != nullptr && weights != nullptr)));
    const uint64_t m = (uint64_t)rows, k = (uint64_t)inputs, n = (uint64_t)outputs, size = type_size(type);
    const uint64_t need = forward_bytes(type, m, k, n), in = m * k * size, w = n * k * size, out = m * n * size;
    DKZ_REQUIRE_WORKSPACE(need);
    const Span writes[] = {{output, out}, {activated, out}, {workspace, need}};
    const Span reads[] = {{input, in}, {weights, w}, {biases, 4 * n}, {residual == output ? nullptr : residual, out}};
    DKZ_REQUIRE(disjoint(writes, reads));
    const Draws draws = make_draws(prob, scale, seed, first);
    const Workspace ws{static_cast<char *>(workspace), need};
    const hipStream_t stream = current_stream();
    // Activations with an exponential are kernels of their own: in one kernel they cost the others too (8192x4096x16384
    // with leaky and dropout 1000 us alone, 1590 beside them).
    return uses_exp(activation)
               ? forward<true>(stream, type, m, k, n, activation, draws, input, weights, biases, residual, activated, output, ws)
               : forward<false>(stream, type, m, k, n, activation, draws, input, weights, biases, residual, activated, output, ws);
}

int dkz_linear_backward_workspace(int type, int rows, int inputs, int outputs, size_t *bytes) {
    DKZ_REQUIRE(bytes != nullptr && type_ok(type) && rows >= 0 && inputs >= 0 && outputs >= 0);
    DKZ_REQUIRE_SIDE(rows);
    DKZ_REQUIRE_SIDE(inputs);
    DKZ_REQUIRE_SIDE(outputs);
    DKZ_REQUIRE_ELEMS(rows, inputs);
    DKZ_REQUIRE_ELEMS(outputs, inputs);
    DKZ_REQUIRE_ELEMS(rows, outputs);
    *bytes = (size_t)backward_plan(type, (uint64_t)rows, (uint64_t)inputs, (uint64_t)outputs).total();
    return 0;
}

int dkz_linear_backward(int type, int rows, int inputs, int outputs, int activation, float prob, float scale, unsigned int seed,
                        unsigned long long first, const void *input, const void *weights, const void *activated,
                        const void *delta, const void *input_residual, float beta, float *bias_updates, void *weight_updates,
                        void *input_delta, void *workspace, size_t workspace_bytes) {
    DKZ_REQUIRE(type_ok(type) && rows >= 0 && inputs >= 0 && outputs >= 0);
    DKZ_REQUIRE(activation >= 0 && activation < kActCount);
    DKZ_REQUIRE_SIDE(rows);
    DKZ_REQUIRE_SIDE(inputs);
    DKZ_REQUIRE_SIDE(outputs);
    DKZ_REQUIRE_ELEMS(rows, inputs);
    DKZ_REQUIRE_ELEMS(outputs, inputs);
    DKZ_REQUIRE_ELEMS(rows, outputs);
    const uint64_t m = (uint64_t)rows, k = (uint64_t)inputs, n = (uint64_t)outputs, size = type_size(type);
    const uint64_t in = m * k * size, w = n * k * size, out = m * n * size;
    const bool products = out != 0 && in + w != 0 && (weight_updates != nullptr || input_delta != nullptr);
    if (out != 0 && (products || bias_updates != nullptr)) {
        DKZ_REQUIRE(delta != nullptr && (activation == kLinear || activated != nullptr));
        DKZ_REQUIRE(in == 0 || weight_updates == nullptr || input != nullptr);
        DKZ_REQUIRE(w == 0 || input_delta == nullptr || weights != nullptr);
    }
    const uint64_t need = backward_plan(type, m, k, n).total();
    DKZ_REQUIRE_WORKSPACE(need);
    const Span writes[] = {{bias_updates, 4 * n}, {weight_updates, w}, {input_delta, in}, {workspace, need}};
    const Span reads[] = {{input, in}, {weights, w}, {activated, out}, {delta, out},
                          {input_residual == input_delta ? nullptr : input_residual, in}};
    DKZ_REQUIRE(disjoint(writes, reads));
    const Draws draws = make_draws(prob, scale, seed, first);
    const Workspace ws{static_cast<char *>(workspace), need};
    const hipStream_t stream = current_stream();
    if (type == DKZ_F32)
        return backward<float>(stream, type, m, k, n, activation, draws, input, weights, activated, delta, input_residual, beta,
                               bias_updates, weight_updates, input_delta, ws);
    return backward<__bf16>(stream, type, m, k, n, activation, draws, input, weights, activated, delta, input_residual, beta,
                            bias_updates, weight_updates, input_delta, ws);
}

}  // extern "C"
