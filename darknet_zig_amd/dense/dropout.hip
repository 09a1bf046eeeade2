// dropout.hip -- dropout whose draws come from a counter, so that no mask or
// draw is stored: y[i] = (draw(seed, first + i) < prob ? 0 : x[i] * scale) +
// residual[i]. The backward pass is the same call on the gradient.
#include "dense_internal.hpp"

namespace dkz {
namespace {

template <class X, class Y>
__device__ __forceinline__ void one(const X *x, const Y *residual, Y *y, uint32_t i, const Draws &draws) {
    const float v = draws.apply(load1(x, i), i);
    store1(y, i, residual != nullptr ? v + load1(residual, i) : v);
}

// Bound by memory. A thread takes eight consecutive elements, kEach times a
// workgroup's width apart, all loads before the first use; the last elements one
// at a time. The two hashes a draw are ~30 instructions an element, less than
// the memory takes: 67 M bf16 elements joined to an fp32 residual 115 us (5.8
// TB/s), 229 us one element a thread.
constexpr uint32_t kEach = 2;

template <class X, class Y>
__global__ __launch_bounds__(kBlock) void dropout_kernel(const X *x, const Y *residual, Y *y, uint32_t n, Draws draws) {
    const uint32_t first = blockIdx.x * (kBlock * kEach) + threadIdx.x;  // in eights
    float v[kEach][8], add[kEach][8] = {};
#pragma unroll
    for (uint32_t u = 0; u < kEach; ++u) {
        const uint32_t i = (first + u * kBlock) * 8;
        if (i + 8 > n) break;
        load8(x, i, v[u]);
        if (residual != nullptr) load8(residual, i, add[u]);
    }
#pragma unroll
    for (uint32_t u = 0; u < kEach; ++u) {
        const uint32_t i = (first + u * kBlock) * 8;
        if (i >= n) break;
        if (i + 8 > n) {
            for (uint32_t e = i; e < n; ++e) one(x, residual, y, e, draws);
            break;
        }
        draws.run(v[u], i);
        if (residual != nullptr) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[u][e] += add[u][e];
        }
        store8(y, i, v[u]);
    }
}

template <class X, class Y>
int run_dropout(const void *x, const void *residual, void *y, uint32_t n, const Draws &draws) {
    const auto *px = static_cast<const X *>(x);
    const auto *pr = static_cast<const Y *>(residual);
    auto *py = static_cast<Y *>(y);
    constexpr const char *kName = "seeded_dropout";
    return launch(kName, dropout_kernel<X, Y>, dim3(div_up(n, 8 * kBlock * kEach)), dim3(kBlock), px, pr, py, n, draws);
}

}  // namespace
}  // namespace dkz

using namespace dkz;

extern "C" int dkz_seeded_dropout(int n, int x_type, const void *x, const void *residual, float prob, float scale,
                                  unsigned int seed, unsigned long long first, int y_type, void *y) {
    DKZ_REQUIRE(n >= 0 && type_ok(x_type) && type_ok(y_type));
    if (n == 0) return 0;
    DKZ_REQUIRE(x != nullptr && y != nullptr);
    const uint64_t xb = (uint64_t)n * type_size(x_type), yb = (uint64_t)n * type_size(y_type);
    DKZ_REQUIRE((x == y && x_type == y_type) || !overlap(x, xb, y, yb));
    DKZ_REQUIRE(residual == y || !overlap(residual, yb, y, yb));
    const Draws draws = make_draws(prob, scale, seed, first);
    if (x_type == DKZ_F32)
        return y_type == DKZ_F32 ? run_dropout<float, float>(x, residual, y, (uint32_t)n, draws)
                                 : run_dropout<float, __bf16>(x, residual, y, (uint32_t)n, draws);
    return y_type == DKZ_F32 ? run_dropout<__bf16, float>(x, residual, y, (uint32_t)n, draws)
                             : run_dropout<__bf16, __bf16>(x, residual, y, (uint32_t)n, draws);
}
