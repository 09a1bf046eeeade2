// dense_internal.hpp -- what the sources of libdkz_dense.so share: the element
// types, the argument checks and the caller's workspace. The stream, the
// sync-after-launch switch and the launch helper are dkz_internal.hpp's, over
// libdkz.so's own state (runtime.hip). The stream is the process's and another host
// thread may set it at any time: an op reads it once and passes it on, so that
// launches that wait for each other are on one stream.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dkz_dense.h"
#include "dkz_device.hpp"
#include "dkz_internal.hpp"

namespace dkz {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// ---- elements: arithmetic is fp32, a bf16 is rounded to nearest even once, as it is stored ----

template <class T>
__device__ __forceinline__ float load1(const T *p, uint64_t i) {
    return (float)p[i];
}
template <class T>
__device__ __forceinline__ void store1(T *p, uint64_t i, float v) {
    p[i] = (T)v;
}
// Eight consecutive elements, at any alignment of theirs (16-byte accesses need none).
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8u __attribute__((ext_vector_type(8), aligned(2)));
template <class T>
__device__ __forceinline__ void load8(const T *p, uint64_t i, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        const f32x4u a = reinterpret_cast<const f32x4u *>(p + i)[0], b = reinterpret_cast<const f32x4u *>(p + i)[1];
#pragma unroll
        for (int x = 0; x < 8; ++x) v[x] = x < 4 ? a[x & 3] : b[x & 3];
    } else {
        const bf16x8u a = *reinterpret_cast<const bf16x8u *>(p + i);
#pragma unroll
        for (int x = 0; x < 8; ++x) v[x] = (float)a[x];
    }
}
template <class T>
__device__ __forceinline__ void store8(T *p, uint64_t i, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<f32x4u *>(p + i)[0] = f32x4u{v[0], v[1], v[2], v[3]};
        reinterpret_cast<f32x4u *>(p + i)[1] = f32x4u{v[4], v[5], v[6], v[7]};
    } else {
        const f32x8 f = {v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]};
        *reinterpret_cast<bf16x8u *>(p + i) = __builtin_convertvector(f, bf16x8);
    }
}

// ---- the elements of a matrix that a thread treats together: N of them, element
// x at index at(x), there if in(x) ----

struct RowRun {  // of one row, next to each other
    uint64_t first;
    uint32_t n;
    static constexpr bool kRow = true;
    __device__ __forceinline__ uint64_t at(int x) const { return first + x; }
    __device__ __forceinline__ bool in(int x) const { return x < (int)n; }
};
struct ColumnRun {  // of one column, in rows next to each other
    uint64_t first;
    uint32_t ld, n;
    static constexpr bool kRow = false;
    __device__ __forceinline__ uint64_t at(int x) const { return first + (uint64_t)x * ld; }
    __device__ __forceinline__ bool in(int x) const { return x < (int)n; }
};
struct BlockColumn {  // of one column, in the rows of a 32x32 block that one lane holds: four, every eight
    uint64_t first;
    uint32_t ld, n;  // n: rows from the first on that exist
    static constexpr bool kRow = false;
    static __device__ __forceinline__ int row(int x) { return (x >> 2) * 8 + (x & 3); }
    __device__ __forceinline__ uint64_t at(int x) const { return first + (uint64_t)row(x) * ld; }
    __device__ __forceinline__ bool in(int x) const { return row(x) < (int)n; }
};

// The elements as they are loaded: kept like this, they are waited for where
// they are used and not where they are loaded.
template <class T, int N>
using Raw = T __attribute__((ext_vector_type(N)));
template <class T, class E, int N>
__device__ __forceinline__ void load_raw(const T *p, const E &e, Raw<T, N> &v) {
    if constexpr (E::kRow && N == 8) {
        if (e.n == 8) {
            if constexpr (sizeof(T) == 4) {
                const f32x4u a = reinterpret_cast<const f32x4u *>(p + e.first)[0], b = reinterpret_cast<const f32x4u *>(p + e.first)[1];
                v = __builtin_shufflevector((f32x4)a, (f32x4)b, 0, 1, 2, 3, 4, 5, 6, 7);
            } else {
                v = *reinterpret_cast<const bf16x8u *>(p + e.first);
            }
            return;
        }
    }
#pragma unroll
    for (int x = 0; x < N; ++x) v[x] = e.in(x) ? p[e.at(x)] : (T)0.0f;
}
template <class T, class E, int N>
__device__ __forceinline__ void store_n(T *p, const E &e, const float (&v)[N]) {
    if constexpr (E::kRow && N == 8) {
        if (e.n == 8) {
            store8(p, e.first, v);
            return;
        }
    }
#pragma unroll
    for (int x = 0; x < N; ++x)
        if (e.in(x)) store1(p, e.at(x), v[x]);
}

inline bool type_ok(int type) { return type == DKZ_F32 || type == DKZ_BF16; }
inline uint64_t type_size(int type) { return type == DKZ_F32 ? 4 : 2; }

// Whether [a, a + an) and [b, b + bn) share a byte; a null pointer shares none.
inline bool overlap(const void *a, uint64_t an, const void *b, uint64_t bn) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return a != nullptr && b != nullptr && an != 0 && bn != 0 && x < y + bn && y < x + an;
}

struct Span {
    const void *p;
    uint64_t bytes;
};
// Whether no span of `writes` shares a byte with one of `reads`, or with another of `writes`.
template <int W, int R>
inline bool disjoint(const Span (&writes)[W], const Span (&reads)[R]) {
    for (int i = 0; i < W; ++i) {
        for (const Span &r : reads)
            if (overlap(writes[i].p, writes[i].bytes, r.p, r.bytes)) return false;
        for (int j = 0; j < i; ++j)
            if (overlap(writes[i].p, writes[i].bytes, writes[j].p, writes[j].bytes)) return false;
    }
    return true;
}

// ---- draws ----

// Element i's draw is the top 24 bits of hash(seed ^ hash(low word of i) ^
// hash(0x9e3779b9 * high word)), times 2^-24; below 2^32 elements, where the
// last hash is 0, it is rand_uniform's. A draw is below prob exactly when its
// 24 bits are below ceil(prob * 2^24) (the host's limit; 0: nothing falls out).
struct Draws {
    uint64_t first;
    uint32_t seed, limit;
    float scale;

    __device__ __forceinline__ bool dropped(uint64_t i) const {
        i += first;
        const uint32_t high = (uint32_t)(i >> 32);
        const uint32_t key = seed ^ (high ? hash_u32(0x9e3779b9u * high) : 0u);
        return hash_u32(key ^ hash_u32((uint32_t)i)) >> 8 < limit;
    }
    // A select, not a multiply: a dropped NaN or infinity is 0.
    __device__ __forceinline__ float apply(float v, uint64_t i) const {
        v *= scale;
        return limit != 0 && dropped(i) ? 0.0f : v;
    }
    template <class E, int N>
    __device__ __forceinline__ void apply(float (&v)[N], const E &e) const {
        if constexpr (E::kRow) {
            run(v, e.first);
        } else {
#pragma unroll
            for (int x = 0; x < N; ++x) v[x] = apply(v[x], e.at(x));
        }
    }
    // Elements i .. i + N - 1.
    template <int N>
    __device__ __forceinline__ void run(float (&v)[N], uint64_t i) const {
#pragma unroll
        for (int x = 0; x < N; ++x) v[x] *= scale;
        if (limit == 0) return;
        i += first;
        const uint32_t low = (uint32_t)i, high = (uint32_t)(i >> 32);
        const uint32_t key = seed ^ (high ? hash_u32(0x9e3779b9u * high) : 0u);
        if (low + (N - 1) >= low) {  // one high word
#pragma unroll
            for (int x = 0; x < N; ++x) v[x] = hash_u32(key ^ hash_u32(low + x)) >> 8 < limit ? 0.0f : v[x];
        } else {
#pragma unroll
            for (int x = 0; x < N; ++x) v[x] = dropped(i - first + x) ? 0.0f : v[x];
        }
    }
};

inline Draws make_draws(float prob, float scale, unsigned int seed, unsigned long long first) {
    // prob * 2^24 is exact in fp32 unless it overflows; a NaN drops nothing, as the comparison with it says.
    const float x = prob * 16777216.0f;
    const uint32_t limit = !(x > 0.0f) ? 0u : x >= 16777216.0f ? 1u << 24 : (uint32_t)x + ((float)(uint32_t)x < x);
    return {first, seed, limit, scale};
}

// ---- the caller's workspace, handed out from its start ----

struct Workspace {
    char *at;
    uint64_t left;

    template <class T>
    T *take(uint64_t n) {
        const uint64_t bytes = (n * sizeof(T) + 255) / 256 * 256;
        if (bytes > left) return nullptr;
        T *p = reinterpret_cast<T *>(at);
        at += bytes;
        left -= bytes;
        return p;
    }
};
inline uint64_t padded(uint64_t bytes) { return (bytes + 255) / 256 * 256; }

inline uint64_t round_up(uint64_t n, uint64_t to) { return (n + to - 1) / to * to; }

}  // namespace dkz

// Matrices past the ABI's largest element count (less what rounds a load up) are refused.
#define DKZ_REQUIRE_ELEMS(a, b) DKZ_REQUIRE((uint64_t)(a) * (uint64_t)(b) + 3 <= kMaxElems)

// A launch counts its threads in 32 bits. Sides up to here keep the kernels that go over rows, columns or a tensor's
// elements below that; products of more workgroups than a launch has room for take several (run_product).
#define DKZ_REQUIRE_SIDE(n) DKZ_REQUIRE((n) <= 1 << 26)

// A call's workspace: `need` bytes at a 16-byte boundary.
#define DKZ_REQUIRE_WORKSPACE(need) \
    DKZ_REQUIRE((need) == 0 || (workspace != nullptr && aligned16(workspace) && workspace_bytes >= (need)))
