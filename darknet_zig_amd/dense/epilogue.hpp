// epilogue.hpp -- what becomes of a product's elements: epilogues of both
// product kernels (put: one element; quad: four of a row), and the column sums
// behind the bias gradients.
#pragma once

#include "dense_internal.hpp"
#include "product.hpp"

namespace dkz {
namespace {

constexpr bool uses_exp(int act) {
    return act == kLogistic || act == kLoggy || act == kElu || act == kSelu || act == kTanh;
}

// The activation `act` of n values: EXP, one of those that take an exponential; else one of the others.
template <bool EXP, int N>
__device__ __forceinline__ void activate_all(int act, float (&x)[N]) {
#define DKZ_ACT(A)                                                      \
    case A:                                                             \
        if constexpr (uses_exp(A) == EXP) {                             \
            _Pragma("unroll") for (int i = 0; i < N; ++i) x[i] = activate<A>(x[i]); \
        }                                                               \
        break;
    switch (act) {
        DKZ_ACT(kLogistic) DKZ_ACT(kRelu) DKZ_ACT(kRelie) DKZ_ACT(kRamp) DKZ_ACT(kTanh) DKZ_ACT(kPlse) DKZ_ACT(kLeaky)
        DKZ_ACT(kElu) DKZ_ACT(kLoggy) DKZ_ACT(kStair) DKZ_ACT(kHardtan) DKZ_ACT(kLhtan) DKZ_ACT(kSelu)
        default: break;
    }
#undef DKZ_ACT
}

// d[i] *= the gradient at the activation's output y[i].
template <int N>
__device__ __forceinline__ void gradient_all(int act, const float (&y)[N], float (&d)[N]) {
#define DKZ_GRAD(A)                                                             \
    case A:                                                                     \
        _Pragma("unroll") for (int i = 0; i < N; ++i) d[i] *= gradient<A>(y[i]); \
        break;
    switch (act) {
        DKZ_GRAD(kLogistic) DKZ_GRAD(kRelu) DKZ_GRAD(kRelie) DKZ_GRAD(kRamp) DKZ_GRAD(kTanh) DKZ_GRAD(kPlse)
        DKZ_GRAD(kLeaky) DKZ_GRAD(kElu) DKZ_GRAD(kLoggy) DKZ_GRAD(kStair) DKZ_GRAD(kHardtan) DKZ_GRAD(kLhtan) DKZ_GRAD(kSelu)
        default: break;
    }
#undef DKZ_GRAD
}

// out = dropout(activation(z + bias)) + residual. Matrices have `ld` columns
// and no gaps, so that r * ld + c is also the draw's element.
template <class T, bool EXP>
struct LinearEpilogue : TileEpilogue<LinearEpilogue<T, EXP>> {
    const float *biases;
    const T *residual;
    T *activated, *output;
    uint32_t ld;
    int act;
    bool vec;
    Draws draws;

    struct Columns {
        float bias[8];
    };
    __device__ __forceinline__ bool whole() const { return vec; }
    __device__ __forceinline__ Columns columns(uint32_t c) const {
        Columns s = {};
        if (vec && biases != nullptr) {
#pragma unroll
            for (int i = 0; i < 8; ++i) s.bias[i] = biases[c + i];
        }
        return s;
    }
    __device__ __forceinline__ void put(uint32_t r, uint32_t c, float z) const {
        const uint64_t at = (uint64_t)r * ld + c;
        float a[1] = {biases != nullptr ? z + biases[c] : z};
        activate_all<EXP>(act, a);
        if (activated != nullptr) store1(activated, at, a[0]);
        draws.apply(a, at);
        store1(output, at, residual != nullptr ? a[0] + load1(residual, at) : a[0]);
    }
    __device__ __forceinline__ void row(const Columns &s, uint32_t r, uint32_t c, float (&a)[8]) const {
        const uint64_t at = (uint64_t)r * ld + c;
        float add[8] = {};
        if (residual != nullptr) load8(residual, at, add);
        if (biases != nullptr) {
#pragma unroll
            for (int i = 0; i < 8; ++i) a[i] += s.bias[i];
        }
        activate_all<EXP>(act, a);
        if (activated != nullptr) store8(activated, at, a);
        draws.apply(a, at);
        if (residual != nullptr) {
#pragma unroll
            for (int i = 0; i < 8; ++i) a[i] += add[i];
        }
        store8(output, at, a);
    }
};

// out = z + beta * old + add, old being out's own value. beta 0 does not read it.
template <class T>
struct StoreEpilogue : TileEpilogue<StoreEpilogue<T>> {
    T *out;
    const T *add;
    uint32_t ld;
    float beta;
    bool vec;

    struct Columns {};
    __device__ __forceinline__ bool whole() const { return vec; }
    __device__ __forceinline__ Columns columns(uint32_t) const { return {}; }
    __device__ __forceinline__ void put(uint32_t r, uint32_t c, float z) const {
        const uint64_t at = (uint64_t)r * ld + c;
        if (beta != 0.0f) z += beta * load1(out, at);
        store1(out, at, add != nullptr ? z + load1(add, at) : z);
    }
    __device__ __forceinline__ void row(const Columns &, uint32_t r, uint32_t c, float (&z)[8]) const {
        const uint64_t at = (uint64_t)r * ld + c;
        float x[8];
        if (beta != 0.0f) {
            load8(out, at, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) z[i] += beta * x[i];
        }
        if (add != nullptr) {
            load8(add, at, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) z[i] += x[i];
        }
        store8(out, at, z);
    }
};

// Whether matrices with rows of ld elements may be moved eight at a time.
inline bool eights(uint64_t ld, const void *a, const void *b = nullptr, const void *c = nullptr) {
    return ld % 8 == 0 && aligned16(a) && aligned16(b) && aligned16(c);
}

template <class T>
StoreEpilogue<T> store_epilogue(void *out, const void *add, uint64_t ld, float beta) {
    StoreEpilogue<T> e;
    e.out = static_cast<T *>(out);
    e.add = static_cast<const T *>(add);
    e.ld = (uint32_t)ld;
    e.beta = beta;
    e.vec = eights(ld, out, add);
    return e;
}

// updates[c] = beta * updates[c] + the sum of column c of partial[chunks][cols],
// in f64: a thread takes every eighth chunk of a column, and a column's eight
// sums are added in order.
__global__ __launch_bounds__(kBlock) void column_sums_kernel(const float *partial, uint32_t chunks, uint32_t cols, float beta,
                                                            float *updates) {
    constexpr uint32_t kLanes = 32, kGroups = kBlock / kLanes;
    __shared__ double sums[kGroups][kLanes];
    const uint32_t x = threadIdx.x % kLanes, group = threadIdx.x / kLanes, c = blockIdx.x * kLanes + x;
    double s = 0.0;
    if (c < cols) {
#pragma unroll 4
        for (uint32_t i = group; i < chunks; i += kGroups) s += (double)partial[(uint64_t)i * cols + c];
    }
    sums[group][x] = s;
    __syncthreads();
    if (group != 0 || c >= cols) return;
#pragma unroll
    for (uint32_t i = 1; i < kGroups; ++i) s += sums[i][x];
    updates[c] = beta == 0.0f ? (float)s : beta * updates[c] + (float)s;
}

inline int add_column_sums(const float *partial, uint64_t chunks, uint64_t cols, float beta, float *updates) {
    if (cols == 0) return 0;
    return launch("bias_updates", column_sums_kernel, dim3(div_up(cols, 32)), dim3(kBlock), partial, (uint32_t)chunks, (uint32_t)cols, beta,
                  updates);
}

}  // namespace
}  // namespace dkz
