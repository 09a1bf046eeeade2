// epilogue.hpp -- what becomes of a product's elements: epilogues of both
// product kernels, and the column sums behind the bias gradients.
#pragma once

#include "dense_internal.hpp"
#include "product.hpp"

namespace dkz {
namespace {

constexpr bool uses_exp(int act) {
    return act == kLogistic || act == kLoggy || act == kElu || act == kSelu || act == kTanh;
}

// An activation with an exponential for a bf16 result: activate<A>'s formula with
// expf_cw, under one ulp of fp32 off, in place of the host's bits, and a
// reciprocal instruction (one ulp) in place of the rounded division: 2^-21
// relative to the larger of 1 and the value, where a bf16 has 2^-9.
template <int A>
__device__ __forceinline__ float activate_bf16(float x) {
    if constexpr (A == kLogistic) return __builtin_amdgcn_rcpf(1.0f + expf_cw(-x));
    else if constexpr (A == kLoggy) return 2.0f * __builtin_amdgcn_rcpf(1.0f + expf_cw(-x)) - 1.0f;
    else if constexpr (A == kElu) return x >= 0.0f ? x : expf_cw(x) - 1.0f;
    else if constexpr (A == kSelu) return x >= 0.0f ? 1.0507f * x : 1.75803124f * (expf_cw(x) - 1.0f);
    else if constexpr (A == kTanh) {
        const float e = expf_cw(2.0f * x);
        return x >= 40.0f ? 1.0f : (e - 1.0f) * __builtin_amdgcn_rcpf(e + 1.0f);  // e is infinite from 44 on
    } else return activate<A>(x);
}

// The activation `act` of N values for a result of type T (fp32 ones are
// activate_array's). EXP: `act` is one of those with an exponential; else one of the others.
template <class T, bool EXP, int N>
__device__ __forceinline__ void activate_all(int act, float (&x)[N]) {
#define DKZ_ACT(A)                                                                                                  \
    case A:                                                                                                         \
        if constexpr (uses_exp(A) == EXP) {                                                                         \
            _Pragma("unroll") for (int i = 0; i < N; ++i)                                                           \
                x[i] = sizeof(T) == 2 ? activate_bf16<A>(x[i]) : activate<A>(x[i]);                                 \
        }                                                                                                           \
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
    bool words;
    Draws draws;

    __device__ __forceinline__ float bias(uint32_t c) const { return biases != nullptr ? biases[c] : 0.0f; }
    __device__ __forceinline__ bool in_words() const { return words; }
    template <int N>
    using Before = Raw<T, N>;
    template <int N, class E>
    __device__ __forceinline__ Before<N> before(const E &e) const {
        Before<N> add = {};
        if (residual != nullptr) load_raw<T, E, N>(residual, e, add);
        return add;
    }
    template <class E, int N>
    __device__ __forceinline__ void put(const E &e, const float (&bias)[N], float (&a)[N], const Before<N> &add) const {
        if (biases != nullptr) {
#pragma unroll
            for (int i = 0; i < N; ++i) a[i] += bias[i];
        }
        activate_all<T, EXP>(act, a);
        if (activated != nullptr) store_n(activated, e, a);
        draws.apply(a, e);
        if (residual != nullptr) {
#pragma unroll
            for (int i = 0; i < N; ++i) a[i] += (float)add[i];
        }
        store_n(output, e, a);
    }
};

// out = alpha * z + beta * old + add, old being out's own value. beta 0 does not read it.
template <class T>
struct StoreEpilogue : TileEpilogue<StoreEpilogue<T>> {
    T *out;
    const T *add;
    uint32_t ld;
    float alpha, beta;
    bool words;

    __device__ __forceinline__ float bias(uint32_t) const { return 0.0f; }
    __device__ __forceinline__ bool in_words() const { return words; }
    template <int N>
    struct Before {
        Raw<T, N> old, add;
    };
    template <int N, class E>
    __device__ __forceinline__ Before<N> before(const E &e) const {
        Before<N> b = {};
        if (beta != 0.0f) load_raw<T, E, N>(out, e, b.old);
        if (add != nullptr) load_raw<T, E, N>(add, e, b.add);
        return b;
    }
    template <class E, int N>
    __device__ __forceinline__ void put(const E &e, const float (&)[N], float (&z)[N], const Before<N> &b) const {
#pragma unroll
        for (int i = 0; i < N; ++i) z[i] *= alpha;
        if (beta != 0.0f) {
#pragma unroll
            for (int i = 0; i < N; ++i) z[i] += beta * (float)b.old[i];
        }
        if (add != nullptr) {
#pragma unroll
            for (int i = 0; i < N; ++i) z[i] += (float)b.add[i];
        }
        store_n(out, e, z);
    }
};

// Whether rows of ld elements of these tensors start on 4-byte boundaries.
template <class T>
bool rows_in_words(uint64_t ld, const void *a, const void *b = nullptr, const void *c = nullptr) {
    return ld * sizeof(T) % 4 == 0 && (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 3) == 0;
}

template <class T>
StoreEpilogue<T> store_epilogue(void *out, const void *add, uint64_t ld, float beta, float alpha = 1.0f) {
    StoreEpilogue<T> e;
    e.out = static_cast<T *>(out);
    e.add = static_cast<const T *>(add);
    e.ld = (uint32_t)ld;
    e.alpha = alpha;
    e.beta = beta;
    e.words = rows_in_words<T>(ld, out, add);
    return e;
}

// updates[c] = beta * updates[c] + the sum of column c of partial[chunks][cols],
// in f64: a thread takes every eighth chunk of a column, and a column's eight
// sums are added in order. `sums` is the workgroup's.
constexpr uint32_t kSumLanes = 32, kSumGroups = kBlock / kSumLanes;
__device__ __forceinline__ void column_sums(const float *partial, uint32_t chunks, uint32_t cols, float beta, float *updates, uint32_t block,
                                            double (&sums)[kSumGroups][kSumLanes]) {
    const uint32_t x = threadIdx.x % kSumLanes, group = threadIdx.x / kSumLanes, c = block * kSumLanes + x;
    double s = 0.0;
    if (c < cols) {
#pragma unroll 4
        for (uint32_t i = group; i < chunks; i += kSumGroups) s += (double)partial[(uint64_t)i * cols + c];
    }
    sums[group][x] = s;
    __syncthreads();
    if (group != 0 || c >= cols) return;
#pragma unroll
    for (uint32_t i = 1; i < kSumGroups; ++i) s += sums[i][x];
    updates[c] = beta == 0.0f ? (float)s : beta * updates[c] + (float)s;
}
__global__ __launch_bounds__(kBlock) void column_sums_kernel(const float *partial, uint32_t chunks, uint32_t cols, float beta,
                                                            float *updates) {
    __shared__ double sums[kSumGroups][kSumLanes];
    column_sums(partial, chunks, cols, beta, updates, blockIdx.x, sums);
}

inline int add_column_sums(hipStream_t stream, const float *partial, uint64_t chunks, uint64_t cols, float beta, float *updates) {
    if (cols == 0) return 0;
    return launch_on(stream, "bias_updates", column_sums_kernel, dim3(div_up(cols, kSumLanes)), dim3(kBlock), partial, (uint32_t)chunks,
                     (uint32_t)cols, beta, updates);
}

}  // namespace
}  // namespace dkz
