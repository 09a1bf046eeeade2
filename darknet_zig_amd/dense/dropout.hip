// dropout.hip -- dropout whose draws come from a counter, so that no mask or
// draw is stored: y[i] = (draw(seed, first + i) < prob ? 0 : x[i] * scale) +
// residual[i]. The backward pass is the same call on the gradient.
#include "dense_internal.hpp"

namespace dkz {
namespace {

template <class X, class Y>
__global__ __launch_bounds__(kBlock) void dropout_kernel(const X *x, const Y *residual, Y *y, uint32_t n, Draws draws) {
    const uint32_t i = blockIdx.x * kBlock + threadIdx.x;
    if (i >= n) return;
    float v = load1(x, i) * draws.scale;
    if (draws.limit != 0 && draws.dropped(i)) v = 0.0f;
    store1(y, i, residual != nullptr ? v + load1(residual, i) : v);
}

template <class X, class Y>
int run_dropout(const void *x, const void *residual, void *y, uint32_t n, const Draws &draws) {
    return launch("seeded_dropout", dropout_kernel<X, Y>, dim3(div_up(n, kBlock)), dim3(kBlock),
                  static_cast<const X *>(x), static_cast<const Y *>(residual), static_cast<Y *>(y), n, draws);
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
