// logits.hpp -- rows of logits: how their kernels share and read them, and the
// sums of a softmax over a row.
//
// A row is read in 16-byte vectors at 16-byte boundaries, whatever its first
// element's address; the vectors at its ends that reach past it are read element
// by element. A group of THREADS threads takes a row, or one of its `parts`; a
// tile is kEach vectors a thread, loaded together.
#pragma once

#include <algorithm>

#include "dense_internal.hpp"
#include "dkz_lm.h"

namespace dkz {
namespace {

__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }

typedef uint32_t u32x4v __attribute__((ext_vector_type(4)));

template <class T>
constexpr uint32_t kVec = 16 / sizeof(T);  // elements of a vector

template <class T>
struct UnalignedOf;
template <>
struct UnalignedOf<float> {
    typedef f32x4u type;
};
template <>
struct UnalignedOf<__bf16> {
    typedef bf16x8u type;
};
template <class T>
using Unaligned = typename UnalignedOf<T>::type;  // a vector at any element

// Logits as the kernels take them.
struct Logits {
    const void *p;
    uint64_t pitch;
    uint32_t rows, classes;
    uint32_t parts, per;  // a row's parts, and the vectors of one
    float inv;            // 1 / temperature
};

// A part of a row: vectors [v0, v1) of 16 bytes from `base`, the row's elements in them being [o, end).
template <class T>
struct Part {
    const T *base;
    uint32_t o, end, v0, v1;

    __device__ __forceinline__ Part(const Logits &g, uint32_t row, uint32_t part) {
        const T *first = static_cast<const T *>(g.p) + (uint64_t)row * g.pitch;
        o = (uint32_t)((uintptr_t)first & 15) / sizeof(T);
        base = first - o;
        end = o + g.classes;
        const uint32_t all = (end + kVec<T> - 1) / kVec<T>;
        v0 = min(part * g.per, all);
        v1 = min(v0 + g.per, all);
    }
    __device__ __forceinline__ bool whole(uint32_t v) const { return v * kVec<T> >= o && (v + 1) * kVec<T> <= end; }
    // Vector v, -infinity in the places outside the row.
    __device__ __forceinline__ u32x4v load(uint32_t v) const {
        if (whole(v)) return *reinterpret_cast<const u32x4v *>(base + (uint64_t)v * kVec<T>);
        Raw<T, kVec<T>> x;
#pragma unroll
        for (uint32_t i = 0; i < kVec<T>; ++i) {
            const uint32_t e = v * kVec<T> + i;
            x[i] = v < v1 && e >= o && e < end ? base[e] : (T)neg_inf();
        }
        return __builtin_bit_cast(u32x4v, x);
    }
    // Whether class c is one of the part's.
    __device__ __forceinline__ bool has(uint32_t c) const { return (o + c) / kVec<T> >= v0 && (o + c) / kVec<T> < v1; }
    // The elements of another tensor's row that are at the places of vector v.
    __device__ __forceinline__ void load_other(const T *row, uint32_t v, float (&x)[kVec<T>]) const {
        if (whole(v)) {
            const auto raw = *reinterpret_cast<const Unaligned<T> *>(row + class_of(v));
#pragma unroll
            for (uint32_t i = 0; i < kVec<T>; ++i) x[i] = (float)raw[i];
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kVec<T>; ++i) {
                const uint32_t e = v * kVec<T> + i;
                x[i] = v < v1 && e >= o && e < end ? load1(row, e - o) : 0.0f;
            }
        }
    }
    __device__ __forceinline__ void store_other(T *row, uint32_t v, const float (&x)[kVec<T>]) const {
        if (whole(v)) {
            Unaligned<T> raw;
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) raw[i] = x[i];
            } else {
                const f32x8 f = {x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]};
                raw = __builtin_convertvector(f, bf16x8);
            }
            *reinterpret_cast<Unaligned<T> *>(row + class_of(v)) = raw;
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kVec<T>; ++i) {
                const uint32_t e = v * kVec<T> + i;
                if (v < v1 && e >= o && e < end) store1(row, e - o, x[i]);
            }
        }
    }
    // The class of vector v's first element; negative, as a 32-bit number, where that lies before the row.
    __device__ __forceinline__ uint32_t class_of(uint32_t v) const { return v * kVec<T> - o; }
};

template <class T>
__device__ __forceinline__ void unpack(const u32x4v &raw, float (&z)[kVec<T>]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t b = raw[i];  // (a bit cast of the vector's element itself gives its first one)
            z[i] = __builtin_bit_cast(float, b);
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            z[2 * i] = __builtin_bit_cast(float, raw[i] << 16);
            z[2 * i + 1] = __builtin_bit_cast(float, raw[i] & 0xffff0000u);
        }
    }
}

// exp(d / temperature) for the elements of a row of T. bf16 logits: the exponential
// instruction on d * (log2(e) / temperature), within |d / temperature| * 2^-23 of it,
// where a step of the logits themselves is 2^-9 of them. fp32: expf_cw, under one ulp.
template <class T>
struct Exp {
    float inv, c;
    __device__ __forceinline__ explicit Exp(float inv) : inv(inv), c(inv * 1.44269504088896341f) {}
    // y in the moment's unit, and exp of it.
    __device__ __forceinline__ float scaled(float d) const { return d * (sizeof(T) == 2 ? c : inv); }
    __device__ __forceinline__ static float of(float y) { return sizeof(T) == 2 ? __builtin_amdgcn_exp2f(y) : expf_cw(y); }
    static constexpr float kUnit = sizeof(T) == 2 ? 0.693147180559945309f : 1.0f;
};

// Of some logits z: their maximum m, and the sums of e = exp((z - m) / T) and of e * (z - m) / T (the latter in
// Exp's unit). Of none: (-infinity, 0, 0). fmaxf passes over NaNs, which stay in the sums.
struct Sums {
    float m, s, t;
};

// What a set's sums are to be multiplied by when the maximum becomes m, and what is added to its (z - m) / T.
// (A finite shift: an empty set's sums are 0, and 0 times infinity is not.)
template <class T>
__device__ __forceinline__ Sums rebased(Sums a, float m, const Exp<T> &ex) {
    const float base = m == neg_inf() ? 0.0f : m;
    const float shift = fmaxf(ex.scaled(a.m - base), -1e30f), f = Exp<T>::of(shift);
    return {m, a.s * f, (a.t + a.s * shift) * f};
}
template <class T>
__device__ __forceinline__ Sums merge(const Sums &a, const Sums &b, const Exp<T> &ex) {
    const float m = fmaxf(a.m, b.m);
    const Sums x = rebased(a, m, ex), y = rebased(b, m, ex);
    return {m, x.s + y.s, x.t + y.t};
}

// Adds U vectors of logits. MOMENT: also their t.
template <class T, bool MOMENT, int U>
__device__ __forceinline__ void add(Sums &a, const u32x4v (&raw)[U], const Exp<T> &ex) {
    float z[U][kVec<T>], m = a.m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        unpack<T>(raw[u], z[u]);
#pragma unroll
        for (uint32_t i = 0; i < kVec<T>; ++i) m = fmaxf(m, z[u][i]);
    }
    const float base = m == neg_inf() ? 0.0f : m;
    a = rebased(a, m, ex);
    float s = 0.0f, t = 0.0f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (uint32_t i = 0; i < kVec<T>; ++i) {
            const float y = ex.scaled(z[u][i] - base), e = Exp<T>::of(y);
            s += e;
            if (MOMENT) t += e * fmaxf(y, -300.0f);  // e is 0 there
        }
    a.s += s;
    a.t += t;
}

// A group's value, in every thread of it. THREADS 64: a wave.
template <class V, int THREADS, class F>
__device__ __forceinline__ V group_reduce(V v, V *lds, F merge_two) {
#pragma unroll
    for (int mask = 1; mask < kWave; mask <<= 1) {
        V o;
        if constexpr (sizeof(V) == 4) {
            o = __shfl_xor(v, mask);
        } else {
            o = {__shfl_xor(v.m, mask), __shfl_xor(v.s, mask), __shfl_xor(v.t, mask)};
        }
        // The lower lane's comes first, so that both lanes have the same bits.
        v = threadIdx.x & mask ? merge_two(o, v) : merge_two(v, o);
    }
    if constexpr (THREADS > kWave) {
        __syncthreads();  // the last use of lds
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = lds[0];
#pragma unroll
        for (int w = 1; w < THREADS / kWave; ++w) v = merge_two(v, lds[w]);
    }
    return v;
}

// log of the sum: of a row without a class left -infinity; NaN stays.
__device__ __forceinline__ float log_sum(const Sums &a) { return a.s == 0.0f ? neg_inf() : logf(a.s); }

// (z - m) / T - l, the log probability of a class. A row without a class left: -infinity.
__device__ __forceinline__ float log_prob_of(float z, float m, float l, float inv) {
    return m == neg_inf() && l == neg_inf() ? neg_inf() : (z - m) * inv - l;
}

// exp(y - l), the probability of a class whose y is in Exp's unit; NaN where l is.
template <class T>
__device__ __forceinline__ float probability(float y, float l) {
    return Exp<T>::of(sizeof(T) == 2 ? y - l * 1.44269504088896341f : y - l);
}

// How rows are shared out: groups of `threads` threads, a row in `parts` of `per` vectors.
struct RowPlan {
    uint32_t threads, parts, per;
    // The workgroups of a launch, which go round the rows' parts.
    uint32_t groups(uint64_t rows) const { return (uint32_t)std::min<uint64_t>(rows * parts, 1u << 20); }
};

constexpr uint32_t kTileVectors = 4;  // vectors a thread and tile
constexpr uint32_t kFill = 512;       // workgroups that are enough for the chip

inline RowPlan plan_rows(int type, uint64_t rows, uint64_t classes) {
    const uint64_t vec = type == DKZ_F32 ? 4 : 8, vectors = (classes + 2 * (vec - 1)) / vec;  // at any alignment
    if (vectors <= kTileVectors * kWave) return {64, 1, (uint32_t)(kTileVectors * kWave)};
    const uint64_t tile = kTileVectors * kBlock, tiles = (vectors + tile - 1) / tile;
    const uint64_t want = std::min<uint64_t>(tiles, rows == 0 ? 1 : (kFill + rows - 1) / rows), each = (tiles + want - 1) / want;
    return {kBlock, (uint32_t)((tiles + each - 1) / each), (uint32_t)(each * tile)};
}

inline Logits make_logits(const RowPlan &plan, const void *p, int rows, int classes, int pitch, float temperature) {
    return {p, (uint64_t)pitch, (uint32_t)rows, (uint32_t)classes, plan.parts, plan.per, 1.0f / temperature};
}

inline bool element_aligned(int type, const void *p) { return (uintptr_t)p % type_size(type) == 0; }

inline bool logits_ok(int type, int rows, int classes, int pitch, float temperature) {
    return type_ok(type) && rows >= 0 && classes >= 0 && pitch >= classes && temperature >= 0x1p-64f && temperature <= 0x1p64f &&
           rows <= 1 << 26 && pitch <= 1 << 26 && (uint64_t)rows * (uint64_t)pitch <= 1ull << 38;
}
// The bytes from a tensor of logits' first element to its last, plus one.
inline uint64_t logits_bytes(int type, int rows, int classes, int pitch) {
    return rows == 0 || classes == 0 ? 0 : ((uint64_t)(rows - 1) * pitch + classes) * type_size(type);
}

}  // namespace
}  // namespace dkz
