// logits.hpp -- rows of logits: how their kernels share and read them, and the
// sums of a softmax over a row.
//
// A row is read in 16-byte vectors at 16-byte boundaries, whatever its first
// element's address; the few elements before and after them (its edges) are taken one
// a thread. A group of THREADS threads takes a row, or one of its `parts`; a
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

// A part of a row: the whole vectors [v0, v1) from `base`, and where it is the row's first or last part the elements before
// the first whole vector or after the last one, its edges: at most kEdges, which the group's first threads take.
template <class T>
struct Part {
    static constexpr uint32_t kEdges = 2 * kVec<T>;
    const T *base;  // the vector that holds the row's first element
    uint32_t o, end, v0, v1;  // the row's elements from base are [o, end)
    bool first, last;

    __device__ __forceinline__ Part(const Logits &g, uint32_t row, uint32_t part) {
        const T *p = static_cast<const T *>(g.p) + (uint64_t)row * g.pitch;
        o = (uint32_t)((uintptr_t)p & 15) / sizeof(T);
        base = p - o;
        end = o + g.classes;
        const uint32_t w0 = o != 0, w1 = max(end / kVec<T>, w0);
        first = part == 0;
        last = part == g.parts - 1;
        v0 = min(w0 + part * g.per, w1);
        v1 = last ? w1 : min(v0 + g.per, w1);
    }
    // Vector v, all of it -infinity past the part's end. (A row is 2^28 bytes at most: a 32-bit offset from an address that
    // all lanes share.)
    __device__ __forceinline__ u32x4v load(uint32_t v) const {
        constexpr uint32_t x = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;
        u32x4v raw = {x, x, x, x};
        if (v < v1) raw = *reinterpret_cast<const u32x4v *>(reinterpret_cast<const char *>(base) + v * 16);
        return raw;
    }
    // Vectors v, v + step ..
    template <int U>
    __device__ __forceinline__ void load(uint32_t v, uint32_t step, u32x4v (&raw)[U]) const {
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = load(v + u * step);
    }
    // The class of vector v's first element.
    __device__ __forceinline__ uint32_t class_of(uint32_t v) const { return v * kVec<T> - o; }
    // The class of this thread's edge, ~0 where it has none.
    __device__ __forceinline__ uint32_t edge() const {
        const uint32_t i = threadIdx.x, w0 = (o != 0) * kVec<T>;  // w0: where the whole vectors begin
        if (first && i < kVec<T> && o + i < min(end, w0)) return i;
        const uint32_t e = max(end / kVec<T> * kVec<T>, w0) + i - kVec<T>;
        return last && i >= kVec<T> && i < kEdges && e < end ? e - o : ~0u;
    }
    // Whether class c is one of the part's.
    __device__ __forceinline__ bool has(uint32_t c) const {
        const uint32_t v = (o + c) / kVec<T>;
        return (v >= v0 || first) && (v < v1 || last);
    }
    // The elements of another tensor's row at the places of vector v.
    __device__ __forceinline__ void load_other(const T *row, uint32_t v, float (&x)[kVec<T>]) const {
        const auto raw = *reinterpret_cast<const Unaligned<T> *>(row + class_of(v));
#pragma unroll
        for (uint32_t i = 0; i < kVec<T>; ++i) x[i] = (float)raw[i];
    }
    __device__ __forceinline__ void store_other(T *row, uint32_t v, const float (&x)[kVec<T>]) const {
        Unaligned<T> raw;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) raw[i] = x[i];
        } else {
            const f32x8 f = {x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]};
            raw = __builtin_convertvector(f, bf16x8);
        }
        *reinterpret_cast<Unaligned<T> *>(row + class_of(v)) = raw;
    }
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

// exp(d / temperature) for the elements of a sum, by the exponential instruction (within a step) on d * (log2(e) / temperature),
// of which three roundings are in the factor and one in the product: off by |d / temperature| * 2^-22 at most, and where d is 0
// not at all.
template <class T>
struct Exp {
    float inv, c;
    __device__ __forceinline__ explicit Exp(float inv) : inv(inv), c(inv * 1.44269504088896341f) {}
    // y in the moment's unit, and exp of it.
    __device__ __forceinline__ float scaled(float d) const { return d * c; }
    __device__ __forceinline__ static float of(float y) { return __builtin_amdgcn_exp2f(y); }
    static constexpr float kUnit = 0.693147180559945309f;
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

// Keeps the compiler from carrying the unpacked logits, twice the registers, from here on.
__device__ __forceinline__ void repacked(u32x4v &raw) { asm volatile("" : "+v"(raw)); }

// The sums of e = exp((z - m) / T) and, MOMENT, e * (z - m) / T over U vectors of logits whose largest is m.
//
// The exponent z * c - m * c is one instruction. m * c is rounded in it, by r, and the sums are multiplied by 2^-r at their
// end: as if it were not. Its products with e are summed as they are, although 0 * -infinity is NaN where a class is masked: then,
// and where m * c is so large that r is no small number, the thread goes through its logits again, each in steps that cannot go
// wrong. (bf16: about 8.5 instead of 12.6 issue slots a logit; 2000 rows of 50001 56.7 -> 50.8 us. fp32, in place of an exponential of under one ulp
// with its own reduction: 1 row of 65536 13.0 -> 11.1 us, 2048 of 65536 105.8 -> 97.1.)
template <class T, bool MOMENT, int U, bool REPACK>
__device__ __forceinline__ Sums sums_from(u32x4v (&raw)[U], float m, const Exp<T> &ex) {
    const float base = m == neg_inf() ? 0.0f : m;
    const auto all = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float z[kVec<T>];
            unpack<T>(raw[u], z);
#pragma unroll
            for (uint32_t i = 0; i < kVec<T>; ++i) f(z[i]);
            if constexpr (REPACK) {
                repacked(raw[u]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    Sums a{m, 0.0f, 0.0f};
    const float mc = base * ex.c;
    all([&](float z) __attribute__((always_inline)) {
        const float y = __builtin_fmaf(z, ex.c, -mc), e = Exp<T>::of(y);
        a.s += e;
        if (MOMENT) a.t = __builtin_fmaf(e, y, a.t);
    });
    const float r = __builtin_fmaf(base, ex.c, -mc), f = Exp<T>::of(-r);
    if (MOMENT) a.t = (a.t - r * a.s) * f;
    a.s *= f;
    if (fabsf(mc) < 0x1p20f && (!MOMENT || a.t == a.t)) return a;
    a.s = a.t = 0.0f;
    all([&](float z) __attribute__((always_inline)) {
        const float y = ex.scaled(z - base), e = Exp<T>::of(y);
        a.s += e;
        if (MOMENT) a.t = __builtin_fmaf(e, fmaxf(y, -300.0f), a.t);  // e is 0 there
    });
    return a;
}

// Adds U vectors of logits, and gives each one's largest. MOMENT: also their t.
template <class T, bool MOMENT, int U>
__device__ __forceinline__ void add(Sums &a, u32x4v (&raw)[U], float (&largest)[U], const Exp<T> &ex) {
    float m = a.m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float z[kVec<T>];
        unpack<T>(raw[u], z);
        largest[u] = z[0];
#pragma unroll
        for (uint32_t i = 1; i < kVec<T>; ++i) largest[u] = fmaxf(largest[u], z[i]);
        m = fmaxf(m, largest[u]);
    }
    a = rebased(a, m, ex);
    const Sums more = sums_from<T, MOMENT, U, false>(raw, m, ex);
    a.s += more.s;
    a.t += more.t;
}
// The same for a wave's vectors v, v + step .. of which only those before `end` are there.
template <class T, bool MOMENT, int U>
__device__ __forceinline__ void add_until(Sums &a, u32x4v (&raw)[U], float (&largest)[U], uint32_t v, uint32_t step, uint32_t end, const Exp<T> &ex) {
    const uint32_t first = __builtin_amdgcn_readfirstlane(v);
    if (first + (U - 1) * step < end) return add<T, MOMENT>(a, raw, largest, ex);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        largest[u] = neg_inf();
        if (first + u * step >= end) continue;
        u32x4v one[1] = {raw[u]};
        float top[1];
        add<T, MOMENT>(a, one, top, ex);
        largest[u] = top[0];
    }
}

// The sums of U vectors of logits that stay packed.
template <class T, int U>
__device__ __forceinline__ Sums sums_of(u32x4v (&raw)[U], const Exp<T> &ex) {
    float m = neg_inf();
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float z[kVec<T>];
        unpack<T>(raw[u], z);
#pragma unroll
        for (uint32_t i = 0; i < kVec<T>; ++i) m = fmaxf(m, z[i]);
        repacked(raw[u]);
        __builtin_amdgcn_sched_barrier(0);
    }
    return sums_from<T, false, U, true>(raw, m, ex);
}

// Adds one logit, -infinity adding nothing.
template <class T>
__device__ __forceinline__ void add_one(Sums &a, float z, const Exp<T> &ex) {
    a = rebased(a, fmaxf(a.m, z), ex);
    const float y = ex.scaled(z - (a.m == neg_inf() ? 0.0f : a.m)), e = Exp<T>::of(y);
    a.s += e;
    a.t += e * fmaxf(y, -300.0f);
}

// The value of lane ^ MASK, without LDS: MASK 1, 2, 3, 7, 8 or 15 within sixteen lanes, 4 as 7 ^ 3, 16 and 32 by the
// instructions that swap rows and halves.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true);
}
template <int MASK>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
    static_assert(MASK == 1 || MASK == 2 || MASK == 3 || MASK == 4 || MASK == 7 || MASK == 8 || MASK == 15 || MASK == 16 || MASK == 31 ||
                  MASK == 32 || MASK == 63, "");
    if constexpr (MASK == 1) return dpp<0xB1>(v);        // quad_perm 1 0 3 2
    else if constexpr (MASK == 2) return dpp<0x4E>(v);   // quad_perm 2 3 0 1
    else if constexpr (MASK == 3) return dpp<0x1B>(v);   // quad_perm 3 2 1 0
    else if constexpr (MASK == 4) return lane_xor<3>(lane_xor<7>(v));
    else if constexpr (MASK == 7) return dpp<0x141>(v);  // row_half_mirror
    else if constexpr (MASK == 8) return dpp<0x128>(v);  // row_ror 8
    else if constexpr (MASK == 15) return dpp<0x140>(v); // row_mirror
    else if constexpr (MASK == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return threadIdx.x & 16 ? r[0] : r[1];
    } else if constexpr (MASK == 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return threadIdx.x & 32 ? r[0] : r[1];
    } else return lane_xor<MASK - 15>(lane_xor<15>(v));  // 31, 63
}
template <>
__device__ __forceinline__ uint32_t lane_xor<63>(uint32_t v) {
    return lane_xor<32>(lane_xor<16>(lane_xor<15>(v)));
}
template <int MASK>
__device__ __forceinline__ float other_lane(float v) {
    return __builtin_bit_cast(float, lane_xor<MASK>(__builtin_bit_cast(uint32_t, v)));
}
template <int MASK>
__device__ __forceinline__ Sums other_lane(const Sums &v) {
    return {other_lane<MASK>(v.m), other_lane<MASK>(v.s), other_lane<MASK>(v.t)};
}

// Joins LANES lanes' values, in all of them. The lower lane's comes first, so that every lane has the same bits. (Groups of
// `mask` lanes have one value, so that mirrors serve as the partners 4 and 8 away.)
template <int LANES, int MASK = 1, class V, class F>
__device__ __forceinline__ V lanes_reduce(V v, F merge_two) {
    if constexpr (MASK < LANES) {
        const V o = other_lane<MASK == 4 ? 7 : MASK == 8 ? 15 : MASK>(v);
        v = threadIdx.x & MASK ? merge_two(o, v) : merge_two(v, o);
        return lanes_reduce<LANES, MASK * 2>(v, merge_two);
    }
    return v;
}
// A group's value, in every thread of it. lds: one a wave.
template <class V, int THREADS, class F>
__device__ __forceinline__ V group_reduce(V v, V *lds, F merge_two) {
    constexpr int kWaves = THREADS / kWave;
    v = lanes_reduce<kWave>(v, merge_two);
    if constexpr (kWaves > 1) {
        __syncthreads();  // the last use of lds
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x / kWave] = v;
        __syncthreads();
        v = lanes_reduce<kWaves>(lds[threadIdx.x % kWaves], merge_two);
    }
    return v;
}

// Of `n` tokens in LDS: whether the jth, which is c, is the first of its class, and the sum of all that class's values, in
// order. (Four are read at once; those past n up to a multiple of four are ~0.)
struct Claim {
    bool first;
    float sum;
};
__device__ __forceinline__ Claim claim(const uint32_t *tokens, const float *values, uint32_t n, uint32_t j, uint32_t c) {
    Claim r{true, 0.0f};
#pragma unroll 4
    for (uint32_t k = 0; k < n; k += 4) {
        const u32x4v token = *reinterpret_cast<const u32x4v *>(tokens + k);
        const float4 value = *reinterpret_cast<const float4 *>(values + k);
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const bool same = token[i] == c;
            r.first &= !(same && k + i < j);
            r.sum += same ? lane(value, (int)i) : 0.0f;
        }
    }
    return r;
}

// log of the sum: of a row without a class left -infinity; NaN stays. The largest logit's own term is 1, but for the rounding that
// sums_from takes out of it again: a sum just below 1 is 1, so that no probability is above it.
__device__ __forceinline__ float log_sum(const Sums &a) { return a.s == 0.0f ? neg_inf() : logf(a.s < 1.0f ? 1.0f : a.s); }

// (z - m) / T - l, the log probability of a class. A row without a class left: -infinity.
__device__ __forceinline__ float log_prob_of(float z, float m, float l, float inv) {
    return m == neg_inf() && l == neg_inf() ? neg_inf() : (z - m) * inv - l;
}

// exp(d / temperature - l), the probability of a class whose logit is d from the largest; NaN where l is. bf16: as the sums'.
// fp32: expf_cw, under one ulp.
template <class T>
__device__ __forceinline__ float probability(float d, float l, const Exp<T> &ex) {
    if constexpr (sizeof(T) == 2) return Exp<T>::of(__builtin_fmaf(d, ex.c, l * -1.44269504088896341f));
    else return expf_cw(d * ex.inv - l);
}

// How rows are shared out: groups of `threads` threads, a row in `parts` of `per` vectors.
struct RowPlan {
    uint32_t threads, parts, per;
    // The workgroups of a launch, which go round the rows' parts.
    uint32_t groups(uint64_t rows) const { return (uint32_t)std::min<uint64_t>(rows * parts, 1u << 20); }
};

constexpr uint32_t kTileVectors = 4;  // vectors a thread and tile
// fill: how many workgroups are to share rows that are too few, a tile each at least.
inline RowPlan plan_rows(int type, uint64_t rows, uint64_t classes, uint64_t fill) {
    const uint64_t vec = type == DKZ_F32 ? 4 : 8, vectors = classes / vec;  // whole ones at most
    if (vectors <= kTileVectors * kWave) return {64, 1, (uint32_t)(kTileVectors * kWave)};
    const uint64_t tile = kTileVectors * kBlock, tiles = (vectors + tile - 1) / tile;
    const uint64_t want = std::min<uint64_t>(tiles, rows == 0 || fill == 0 ? 1 : fill / rows + (fill % rows != 0)), each = (tiles + want - 1) / want;
    return {kBlock, (uint32_t)((tiles + each - 1) / each), (uint32_t)(each * tile)};
}
// Where the parts' results are joined by another launch, which takes as long as three tiles: parts where they save more. (fp32, top
// 20, us in parts and in one: 1 row of 2 tiles 11.7 and 8.8, of 4 11.9 and 12.2, of 5 12.3 and 13.6; 200 rows of 5 20.0 and 17.2.
// bf16, top 5, 7 tiles: 200 rows 19.1 and 20.1, 300 rows 23.5 and 21.7.)
constexpr uint64_t kJoinFill = 512;
inline RowPlan plan_joined_rows(int type, uint64_t rows, uint64_t classes) {
    constexpr uint64_t kJoinTiles = 3;
    const uint64_t tile = kTileVectors * kBlock * (type == DKZ_F32 ? 4 : 8), tiles = (classes + tile - 1) / tile;
    return plan_rows(type, rows, classes, kJoinTiles + (tiles * rows + kJoinFill - 1) / kJoinFill < tiles ? kJoinFill : 0);
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
