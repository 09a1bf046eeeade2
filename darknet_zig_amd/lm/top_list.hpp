// top_list.hpp -- the largest logits that a wave has seen, in order, one a lane.
//
// A logit and its class are one 64-bit key: the logit's bits in an order of unsigned
// integers, then the class's complement, so that of equal logits the lowest class is
// the largest key. No key is 0.
#pragma once

#include "logits.hpp"

namespace dkz {
namespace {

constexpr int kMostTop = kWave;

// A logit in the order of unsigned integers: a NaN above all, -0 as +0.
__device__ __forceinline__ uint32_t ordered(float z) {
    const uint32_t b = __builtin_bit_cast(uint32_t, z + 0.0f);
    return z != z ? 0xffffffffu : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t order) {
    return __builtin_bit_cast(float, order ^ (order >> 31 ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t key_of(float z, uint32_t c) { return (uint64_t)ordered(z) << 32 | (uint32_t)~c; }
constexpr uint64_t kMaskedKey = (uint64_t)0x007fffffu << 32 | 0xffffffffu;  // no key of -infinity is above it

__device__ __forceinline__ uint64_t from_lane(uint64_t v, int mask) {
    return (uint64_t)(uint32_t)__shfl_xor((int)(uint32_t)(v >> 32), mask) << 32 | (uint32_t)__shfl_xor((int)(uint32_t)v, mask);
}

// One step of a bitonic network: lanes without bit `bit` keep the larger of theirs and their partner's (`mask` away).
template <class V, class X>
__device__ __forceinline__ V exchange(V v, int mask, int bit, X partner) {
    const V o = partner(v, mask);
    const bool larger = (threadIdx.x & bit) == 0;
    return (o > v) == larger ? o : v;
}
// A wave's values in descending order.
template <class V, class X>
__device__ __forceinline__ V sorted(V v, X partner) {
#pragma unroll
    for (int size = 2; size <= kWave; size <<= 1) {
        v = exchange(v, size - 1, size >> 1, partner);
#pragma unroll
        for (int step = size >> 2; step > 0; step >>= 1) v = exchange(v, step, step, partner);
    }
    return v;
}
// The largest 64 of two descending sequences, the second given from its end (lane i has its element 63 - i).
__device__ __forceinline__ uint64_t merged(uint64_t a, uint64_t b_reversed) {
    uint64_t v = a > b_reversed ? a : b_reversed;
#pragma unroll
    for (int step = kWave / 2; step > 0; step >>= 1) v = exchange(v, step, step, from_lane);
    return v;
}

// A wave's list and the candidates that wait to be merged into it, in LDS.
struct TopList {
    static constexpr int kRoom = 2 * kWave;
    uint64_t list = 0;   // lane i: the (i + 1)th largest key, 0 where there are fewer
    uint64_t least;      // a candidate's key is above it
    uint64_t *waiting;   // [kRoom], this wave's
    uint32_t count = 0, top;

    __device__ __forceinline__ TopList(uint64_t *waiting, uint32_t top) : least(kMaskedKey), waiting(waiting), top(top) {}

    __device__ __forceinline__ static uint32_t lane() { return threadIdx.x & 63; }
    __device__ __forceinline__ static void fence() {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }

    // Keys above `least` (those of -infinity are not) are candidates.
    __device__ __forceinline__ void offer(uint64_t key) {
        const bool in = key > least;
        const uint64_t lanes = __ballot(in);
        if (lanes == 0) return;
        if (in) waiting[count + __popcll(lanes & ((1ull << lane()) - 1))] = key;
        count += (uint32_t)__popcll(lanes);
        if (count >= kWave) flush();
    }
    // Merges the first 64 that wait, or all.
    __device__ __forceinline__ void flush() {
        fence();
        const uint32_t n = min(count, (uint32_t)kWave);
        uint64_t key = lane() < n ? waiting[lane()] : 0, rest = kWave + lane() < count ? waiting[kWave + lane()] : 0;
        fence();
        if (count > kWave && kWave + lane() < count) waiting[lane()] = rest;
        count -= n;
        key = sorted(key, from_lane);
        list = merged(list, from_lane(key, kWave - 1));
        const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(list >> 32), (int)top - 1);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)list, (int)top - 1);
        const uint64_t last = (uint64_t)hi << 32 | lo;
        if (last > least) least = last;
    }
    __device__ __forceinline__ void finish() {
        if (count > 0) flush();
    }
};

}  // namespace
}  // namespace dkz
