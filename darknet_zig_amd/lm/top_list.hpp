// top_list.hpp -- the largest logits that a wave has seen, in order, one a lane.
//
// A logit and its class are one 64-bit key: the logit's bits in an order of unsigned
// integers, then the class's complement, so that of equal logits the lowest class is
// the largest key. No key is 0. (Keys of NaNs are not looked at: their row has no
// alternatives.)
//
// A row is gone through once. A lower bound on the last of the list keeps nearly all of
// a row out: the vectors that hold a larger logit (the softmax needs every vector's
// largest anyway) are collected in LDS, their logits above the bound wait there, and
// 64 of them are sorted and merged into the list at once, which raises the bound. The
// first bound is the `top`th of the lanes' largest logits of their first tile.
#pragma once

#include "logits.hpp"

namespace dkz {
namespace {

constexpr int kMostTop = kWave;

// A logit in the order of unsigned integers, -0 as +0.
__device__ __forceinline__ uint32_t ordered(float z) {
    const uint32_t b = __builtin_bit_cast(uint32_t, z + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t order) {
    return __builtin_bit_cast(float, order ^ (order >> 31 ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t key_of(float z, uint32_t c) { return (uint64_t)ordered(z) << 32 | (uint32_t)~c; }
constexpr uint32_t kMaskedOrder = 0x007fffffu;  // of -infinity

template <int MASK>
__device__ __forceinline__ uint64_t lane_xor(uint64_t v) {
    return (uint64_t)lane_xor<MASK>((uint32_t)(v >> 32)) << 32 | lane_xor<MASK>((uint32_t)v);
}

// One step of a bitonic network: lanes without bit BIT keep the larger of theirs and lane ^ MASK's.
template <int MASK, int BIT, class V>
__device__ __forceinline__ V exchange(V v) {
    const V o = lane_xor<MASK>(v);
    const bool larger = (threadIdx.x & BIT) == 0;
    return (o > v) == larger ? o : v;
}
// Descending, given that the lanes' first and second half of 2 * STEP are one up and one down.
template <int STEP, class V>
__device__ __forceinline__ V untangled(V v) {
    if constexpr (STEP > 0) return untangled<STEP / 2>(exchange<STEP, STEP>(v));
    else return v;
}
// A wave's values in descending order; those from lane n on are 0.
template <int SIZE = 2, class V>
__device__ __forceinline__ V sorted(V v, uint32_t n = kWave) {
    if (SIZE > 16 && n <= SIZE / 2) return v;  // the last stages would move zeros
    v = untangled<SIZE / 4>(exchange<SIZE - 1, SIZE / 2>(v));
    if constexpr (SIZE < kWave) return sorted<SIZE * 2>(v, n);
    else return v;
}
// The largest 64 of two descending sequences, the second given from its end (lane i has its element 63 - i).
__device__ __forceinline__ uint64_t merged(uint64_t a, uint64_t b_reversed) {
    return untangled<kWave / 2>(a > b_reversed ? a : b_reversed);
}

// What a wave's list keeps in LDS.
struct TopRoom {
    u32x4v vectors[kTileVectors * kWave];  // a tile's that hold a candidate
    uint32_t classes[kTileVectors * kWave];  // their first elements'
    uint64_t waiting[2 * kWave];
};

template <class T>
struct TopList {
    TopRoom &room;
    uint64_t list = 0;  // lane i: the (i + 1)th largest key, 0 where there are fewer
    uint64_t least;     // a candidate's key is above it
    float bound;        // and its logit at least this
    uint32_t count = 0, top;
    bool any = false;  // whether the list has been merged into

    __device__ __forceinline__ TopList(TopRoom &room, uint32_t top) : room(room), top(top) { raise(kMaskedOrder, 0xffffffffu); }

    __device__ __forceinline__ static uint32_t lane() { return threadIdx.x & 63; }
    __device__ __forceinline__ static uint32_t before(uint64_t lanes) { return (uint32_t)__popcll(lanes & ((1ull << lane()) - 1)); }
    __device__ __forceinline__ static void fence() {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    // Later classes whose logit is the bound's own come after those of the list: only larger logits are of interest.
    __device__ __forceinline__ void raise(uint32_t order, uint32_t low) {
        least = (uint64_t)order << 32 | low;
        bound = logit_of(order + 1);
    }

    // The first tile: a list's last is at least the `top`th of the lanes' largest logits.
    __device__ __forceinline__ void begin(float largest) {
        const uint32_t order = (uint32_t)__builtin_amdgcn_readlane((int)sorted(ordered(largest)), (int)top - 1);
        if (order <= kMaskedOrder) return;
        least = (uint64_t)order << 32;
        bound = logit_of(order);
    }
    // A tile of vectors, vector u's first class being first_class(u).
    template <int U, class F>
    __device__ __forceinline__ void tile(const u32x4v (&raw)[U], const float (&largest)[U], F first_class) {
        uint32_t n = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool in = largest[u] >= bound;
            const uint64_t lanes = __ballot(in);
            if (lanes == 0) continue;
            if (in) {
                const uint32_t at = n + before(lanes);
                room.vectors[at] = raw[u];
                room.classes[at] = first_class(u);
            }
            n += (uint32_t)__popcll(lanes);
        }
        if (n == 0) return;
        fence();
#pragma unroll 1
        for (uint32_t e0 = 0; e0 < n * kVec<T>; e0 += kWave) {
            const uint32_t e = e0 + lane(), v = min(e / kVec<T>, n - 1);
            const float z = load1(reinterpret_cast<const T *>(room.vectors), min(e, n * kVec<T> - 1));
            offer(e < n * kVec<T> ? key_of(z, room.classes[v] + e % kVec<T>) : 0);
        }
        fence();
    }
    __device__ __forceinline__ void offer(uint64_t key) {
        const bool in = key > least;
        const uint64_t lanes = __ballot(in);
        if (in) room.waiting[count + before(lanes)] = key;
        count += (uint32_t)__popcll(lanes);
        if (count >= kWave) flush();
    }
    // Merges the first 64 that wait, or all.
    __device__ __forceinline__ void flush() {
        fence();
        const uint32_t n = min(count, (uint32_t)kWave);
        const uint64_t key = lane() < n ? room.waiting[lane()] : 0, rest = room.waiting[kWave + lane()];
        fence();
        if (kWave + lane() < count) room.waiting[lane()] = rest;
        count -= n;
        const uint64_t more = sorted(key, n);
        list = any ? merged(list, lane_xor<kWave - 1>(more)) : more;
        any = true;
        const uint32_t order = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(list >> 32), (int)top - 1);
        const uint32_t low = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)list, (int)top - 1);
        if (((uint64_t)order << 32 | low) > least) raise(order, low);
    }
    __device__ __forceinline__ void finish() {
        if (count > 0) flush();
    }
};

}  // namespace
}  // namespace dkz
