// token_log_probs.hip -- log probabilities of given tokens, the entropy and the top
// alternatives from a row of logits, and the delta of the logits from theirs.
#include "logits.hpp"
#include "top_list.hpp"

namespace dkz {
namespace {

constexpr int kMostGiven = 256;

struct Answers {
    const int *tokens;
    float *log_probs, *entropy, *stats;
    int *top_tokens;
    float *top_log_probs;
    uint32_t given, top;
    // Of rows in several parts: [rows * parts], and [rows * parts][top].
    Sums *part_sums;
    uint64_t *part_keys;
};

// What a row's group writes, all of its threads having the row's sums and the first wave its list.
template <class T, int THREADS>
struct Answer {
    static constexpr int kSlots = kMostGiven / THREADS;
    uint32_t token[kSlots];
    float z[kSlots];

    // The given tokens and their logits, ahead of the row's sums.
    __device__ __forceinline__ void begin(const Logits &g, const Answers &out, uint32_t row) {
        const T *logits = static_cast<const T *>(g.p) + (uint64_t)row * g.pitch;
#pragma unroll
        for (int i = 0; i < kSlots; ++i) {
            const uint32_t j = threadIdx.x + i * THREADS;
            token[i] = j < out.given ? (uint32_t)out.tokens[(uint64_t)row * out.given + j] : ~0u;
        }
#pragma unroll
        for (int i = 0; i < kSlots; ++i) z[i] = token[i] < g.classes ? load1(logits, token[i]) : 0.0f;
    }
    __device__ __forceinline__ void finish(const Logits &g, const Answers &out, uint32_t row, const Sums &a, uint64_t list) const {
        const float l = log_sum(a);
        if (threadIdx.x == 0) {
            out.stats[2 * (uint64_t)row] = a.m;
            out.stats[2 * (uint64_t)row + 1] = l;
            // l and -t / s are both at least 0, the latter but for its rounding: nothing cancels. NaN stays.
            if (out.entropy != nullptr) {
                const float h = l - Exp<T>::kUnit * (a.t / a.s);
                out.entropy[row] = a.s == 0.0f || h < 0.0f ? 0.0f : h;
            }
        }
#pragma unroll
        for (int i = 0; i < kSlots; ++i) {
            const uint32_t j = threadIdx.x + i * THREADS;
            if (j < out.given) out.log_probs[(uint64_t)row * out.given + j] = token[i] < g.classes ? log_prob_of(z[i], a.m, l, g.inv) : 0.0f;
        }
        if (threadIdx.x < out.top) {
            const uint64_t at = (uint64_t)row * out.top + threadIdx.x;
            const bool has = list != 0 && l == l;
            out.top_tokens[at] = has ? (int)~(uint32_t)list : -1;
            out.top_log_probs[at] = has ? log_prob_of(logit_of((uint32_t)(list >> 32)), a.m, l, g.inv) : l == l ? neg_inf() : l;
        }
    }
};

// The waves' lists joined two and two, in the first wave. keys: one a thread.
template <int WAVES>
__device__ __forceinline__ uint64_t join_lists(uint64_t list, uint64_t *keys) {
    const uint32_t wave = threadIdx.x / kWave, lane = threadIdx.x & 63;
#pragma unroll
    for (uint32_t step = 1; step < WAVES; step *= 2) {
        if (wave % (2 * step) == step) keys[threadIdx.x] = list;
        __syncthreads();
        if (wave % (2 * step) == 0) list = merged(list, keys[(wave + step) * kWave + kWave - 1 - lane]);
    }
    return list;
}

// A group takes a part of a row: its sums in one pass, and its list of the largest.
template <class T, int THREADS, bool ENTROPY, bool TOP>
__global__ __launch_bounds__(THREADS) void log_probs_kernel(Logits g, Answers out) {
    constexpr int kEach = kTileVectors, kWaves = THREADS / kWave;
    __shared__ Sums lds[kWaves];
    __shared__ TopRoom rooms[TOP ? kWaves : 1];
    __shared__ uint64_t keys[TOP ? THREADS : 1];
    const Exp<T> ex(g.inv);
    for (uint32_t group = blockIdx.x; group < g.rows * g.parts; group += gridDim.x) {
        const uint32_t row = group / g.parts, part = group - row * g.parts;
        const Part<T> p(g, row, part);
        Answer<T, THREADS> answer;
        if (g.parts == 1) answer.begin(g, out, row);
        const uint32_t edge = p.edge();
        const float at_edge = edge != ~0u ? load1(static_cast<const T *>(g.p) + (uint64_t)row * g.pitch, edge) : neg_inf();
        Sums a{neg_inf(), 0.0f, 0.0f};
        TopList<T> top(rooms[TOP ? threadIdx.x / kWave : 0], TOP ? out.top : 1);
        for (uint32_t v0 = p.v0 + threadIdx.x; v0 - threadIdx.x < p.v1; v0 += kEach * THREADS) {
            u32x4v raw[kEach];
            float largest[kEach];
            p.load(v0, THREADS, raw);
            add_until<T, ENTROPY>(a, raw, largest, v0, THREADS, p.v1, ex);
            if constexpr (TOP) {
                if (v0 - threadIdx.x == p.v0) top.begin(a.m);
                top.tile(raw, largest, [&](int u) { return p.class_of(v0 + u * THREADS); });
            }
        }
        add_one(a, at_edge, ex);
        a = group_reduce<Sums, THREADS>(a, lds, [&](const Sums &x, const Sums &y) { return merge(x, y, ex); });
        uint64_t list = 0;
        if constexpr (TOP) {
            top.offer(edge != ~0u ? key_of(at_edge, edge) : 0);
            top.finish();
            list = join_lists<kWaves>(top.list, keys);
        }
        if (g.parts == 1) {
            answer.finish(g, out, row, a, list);
        } else {
            if (threadIdx.x == 0) out.part_sums[group] = a;
            if (TOP && threadIdx.x < out.top) out.part_keys[(uint64_t)group * out.top + threadIdx.x] = list;
        }
        if (TOP && kWaves > 1) __syncthreads();  // the keys' use
    }
}

// Joins a row's parts, a group of 256 threads a row.
template <class T, bool TOP>
__global__ __launch_bounds__(kBlock) void join_log_probs_kernel(Logits g, Answers out) {
    constexpr int kWaves = kBlock / kWave, kAhead = 4;
    __shared__ Sums lds[kWaves];
    __shared__ uint64_t keys[TOP ? kBlock : 1];
    const Exp<T> ex(g.inv);
    const uint32_t row = blockIdx.x, wave = threadIdx.x / kWave, back = kWave - 1 - (threadIdx.x & 63);
    Answer<T, kBlock> answer;
    answer.begin(g, out, row);
    // A wave's lists, loaded a few at a time and from their ends.
    const auto load = [&](uint64_t(&next)[kAhead], uint32_t p0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const uint32_t p = p0 + i * kWaves;
            const uint32_t at = i == 0 && p0 == wave ? kWave - 1 - back : back;  // the first one is the list to begin with
            next[i] = p < g.parts && at < out.top ? out.part_keys[((uint64_t)row * g.parts + p) * out.top + at] : 0;
        }
    };
    uint64_t list = 0, next[kAhead];
    if constexpr (TOP) load(next, wave);
    Sums a{neg_inf(), 0.0f, 0.0f};
    for (uint32_t p = threadIdx.x; p < g.parts; p += kBlock) a = merge(a, out.part_sums[(uint64_t)row * g.parts + p], ex);
    a = group_reduce<Sums, kBlock>(a, lds, [&](const Sums &x, const Sums &y) { return merge(x, y, ex); });
    if constexpr (TOP) {
        for (uint32_t p = wave; p < g.parts; p += kAhead * kWaves) {
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                if (i == 0 && p == wave) list = next[0];
                else if (p + i * kWaves < g.parts) list = merged(list, next[i]);
            }
            load(next, p + kAhead * kWaves);
        }
        list = join_lists<kWaves>(list, keys);
    }
    answer.finish(g, out, row, a, list);
}

uint64_t part_bytes(uint64_t rows, const RowPlan &p, uint64_t top) {
    return p.parts == 1 ? 0 : padded(rows * p.parts * sizeof(Sums)) + padded(rows * p.parts * top * 8);
}
// The most that any number of rows up to `rows` takes: from kJoinFill on they have no parts.
uint64_t most_part_bytes(int type, uint64_t rows, uint64_t classes, uint64_t top) {
    uint64_t most = 0;
    for (uint64_t r = 1; r <= std::min(rows, kJoinFill); ++r) most = std::max(most, part_bytes(r, plan_joined_rows(type, r, classes), top));
    return most;
}

template <class T, bool ENTROPY, bool TOP>
int run_log_probs(hipStream_t stream, const Logits &g, const RowPlan &plan, const Answers &out) {
    constexpr const char *kName = "token_log_probs";
    const dim3 grid(plan.groups(g.rows));
    if (plan.threads == 64) return launch_on(stream, kName, log_probs_kernel<T, 64, ENTROPY, TOP>, grid, dim3(64), g, out);
    DKZ_TRY(launch_on(stream, kName, log_probs_kernel<T, kBlock, ENTROPY, TOP>, grid, dim3(kBlock), g, out));
    if (plan.parts == 1) return 0;
    return launch_on(stream, "token_log_probs_join", join_log_probs_kernel<T, TOP>, dim3(g.rows), dim3(kBlock), g, out);
}

template <class T>
int log_probs(hipStream_t stream, const Logits &g, const RowPlan &plan, const Answers &out) {
    if (out.top != 0) return out.entropy != nullptr ? run_log_probs<T, true, true>(stream, g, plan, out) : run_log_probs<T, false, true>(stream, g, plan, out);
    return out.entropy != nullptr ? run_log_probs<T, true, false>(stream, g, plan, out) : run_log_probs<T, false, false>(stream, g, plan, out);
}

// ---- backward ----

struct Deltas {
    const int *tokens;
    const float *stats, *entropy, *a, *e;
    void *out;
    float beta;
    uint32_t given;
};

// A group takes a part of a row. The tokens' classes are written a second time, when
// the others have been, by the thread that has a class's first token.
template <class T, int THREADS, bool ENTROPY, bool OLD>
__global__ __launch_bounds__(THREADS) void log_probs_backward_kernel(Logits g, Deltas in) {
    constexpr int kEach = kTileVectors;
    __shared__ float sums[THREADS / kWave];
    __shared__ __align__(16) uint32_t tokens[kMostGiven];
    __shared__ __align__(16) float deltas[kMostGiven];
    const Exp<T> ex(g.inv);
    for (uint32_t group = blockIdx.x; group < g.rows * g.parts; group += gridDim.x) {
        const uint32_t row = group / g.parts, part = group - row * g.parts;
        const Part<T> p(g, row, part);
        T *out = static_cast<T *>(in.out) + (uint64_t)row * g.pitch;
        const T *logits = static_cast<const T *>(g.p) + (uint64_t)row * g.pitch;
        const float m = in.stats[2 * (uint64_t)row], l = in.stats[2 * (uint64_t)row + 1];
        const bool none = m == neg_inf() && l == neg_inf();
        const float e = ENTROPY ? in.e[row] : 0.0f, h = ENTROPY ? in.entropy[row] : 0.0f;

        __syncthreads();
        float total = 0.0f;
        for (uint32_t j = threadIdx.x; j < (in.given + 3) / 4 * 4; j += THREADS) {
            const uint32_t c = j < in.given ? (uint32_t)in.tokens[(uint64_t)row * in.given + j] : ~0u;
            const float a = c < g.classes ? in.a[(uint64_t)row * in.given + j] : 0.0f;
            tokens[j] = c;
            deltas[j] = a;
            total += a;
        }
        total = group_reduce<float, THREADS>(total, sums, [](float x, float y) { return x + y; });
        __syncthreads();
        // p * (A + e * (log p + H)) / T
        const auto dense = [&](float z) __attribute__((always_inline)) {
            const float y = ex.scaled(z - m), log_p = Exp<T>::kUnit * fmaxf(y, -300.0f) - l;
            const float q = ENTROPY ? total + e * (log_p + h) : total;
            return none ? 0.0f : -(probability<T>(z - m, l, ex) * q) * g.inv;
        };
        constexpr int kSlots = kMostGiven / THREADS > 1 ? kMostGiven / THREADS : 1;
        float fixed[kSlots];
        bool mine[kSlots];
#pragma unroll
        for (int i = 0; i < kSlots; ++i) {
            const uint32_t j = threadIdx.x + i * THREADS;
            mine[i] = false;
            if (j >= in.given) continue;
            const uint32_t c = tokens[j];
            if (c >= g.classes || !p.has(c)) continue;
            const Claim own = claim(tokens, deltas, in.given, j, c);
            mine[i] = own.first;
            fixed[i] = dense(load1(logits, c)) + (none ? 0.0f : own.sum * g.inv);
            if (OLD) fixed[i] += in.beta * load1(out, c);
        }
        __syncthreads();  // what logits_delta's old values, or the logits in its place, have been read for
        for (uint32_t v0 = p.v0; v0 < p.v1; v0 += kEach * THREADS) {
            u32x4v raw[kEach];
            float old[OLD ? kEach : 1][kVec<T>];
            p.load(v0 + threadIdx.x, THREADS, raw);
            if constexpr (OLD) {
#pragma unroll
                for (int u = 0; u < kEach; ++u)
                    if (v0 + u * THREADS + threadIdx.x < p.v1) p.load_other(out, v0 + u * THREADS + threadIdx.x, old[u]);
            }
#pragma unroll
            for (int u = 0; u < kEach; ++u) {
                float z[kVec<T>];
                unpack<T>(raw[u], z);
#pragma unroll
                for (uint32_t i = 0; i < kVec<T>; ++i) {
                    z[i] = dense(z[i]);
                    if constexpr (OLD) z[i] += in.beta * old[u][i];
                }
                if (v0 + u * THREADS + threadIdx.x < p.v1) p.store_other(out, v0 + u * THREADS + threadIdx.x, z);
            }
        }
        if (const uint32_t c = p.edge(); c != ~0u) store1(out, c, dense(load1(logits, c)) + (OLD ? in.beta * load1(out, c) : 0.0f));
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kSlots; ++i)
            if (mine[i]) store1(out, tokens[threadIdx.x + i * THREADS], fixed[i]);
    }
}

template <class T, int THREADS>
int run_backward(hipStream_t stream, const Logits &g, const RowPlan &plan, const Deltas &in) {
    constexpr const char *kName = "token_log_probs_backward";
    const dim3 grid(plan.groups(g.rows)), block(THREADS);
    if (in.e != nullptr)
        return in.beta != 0.0f ? launch_on(stream, kName, log_probs_backward_kernel<T, THREADS, true, true>, grid, block, g, in)
                               : launch_on(stream, kName, log_probs_backward_kernel<T, THREADS, true, false>, grid, block, g, in);
    return in.beta != 0.0f ? launch_on(stream, kName, log_probs_backward_kernel<T, THREADS, false, true>, grid, block, g, in)
                           : launch_on(stream, kName, log_probs_backward_kernel<T, THREADS, false, false>, grid, block, g, in);
}

}  // namespace
}  // namespace dkz

using namespace dkz;

extern "C" {

int dkz_token_log_probs_workspace(int type, int rows, int classes, int top, size_t *bytes) {
    DKZ_REQUIRE(bytes != nullptr && logits_ok(type, rows, classes, classes, 1.0f) && top >= 0 && top <= kMostTop);
    *bytes = (size_t)most_part_bytes(type, (uint64_t)rows, (uint64_t)classes, (uint64_t)top);
    return 0;
}

int dkz_token_log_probs(int type, int rows, int classes, int pitch, const void *logits, float temperature, int given,
                        const int *tokens, int top, float *log_probs_out, float *entropy, float *stats, int *top_tokens,
                        float *top_log_probs, void *workspace, size_t workspace_bytes) {
    DKZ_REQUIRE(logits_ok(type, rows, classes, pitch, temperature));
    DKZ_REQUIRE(given >= 0 && given <= kMostGiven && top >= 0 && top <= kMostTop);
    if (rows == 0) return 0;
    const uint64_t m = (uint64_t)rows, n = m * (uint64_t)given, k = m * (uint64_t)top;
    DKZ_REQUIRE(stats != nullptr && (classes == 0 || logits != nullptr));
    DKZ_REQUIRE(given == 0 || (tokens != nullptr && log_probs_out != nullptr));
    DKZ_REQUIRE(top == 0 || (top_tokens != nullptr && top_log_probs != nullptr));
    const RowPlan plan = plan_joined_rows(type, rows, classes);
    const uint64_t need = part_bytes(m, plan, (uint64_t)top);
    DKZ_REQUIRE_WORKSPACE(need);
    DKZ_REQUIRE(element_aligned(type, logits));
    const Span writes[] = {{log_probs_out, 4 * n}, {entropy, 4 * m}, {stats, 8 * m}, {top_tokens, 4 * k}, {top_log_probs, 4 * k}, {workspace, need}};
    const Span reads[] = {{logits, logits_bytes(type, rows, classes, pitch)}, {tokens, 4 * n}};
    DKZ_REQUIRE(disjoint(writes, reads));
    Workspace ws{static_cast<char *>(workspace), need};
    Answers out{tokens, log_probs_out, entropy, stats, top_tokens, top_log_probs, (uint32_t)given, (uint32_t)top, nullptr, nullptr};
    if (plan.parts > 1) {
        out.part_sums = ws.take<Sums>(m * plan.parts);
        out.part_keys = ws.take<uint64_t>(m * plan.parts * (uint64_t)top);
    }
    const Logits g = make_logits(plan, logits, rows, classes, pitch, temperature);
    const hipStream_t stream = current_stream();
    return type == DKZ_F32 ? log_probs<float>(stream, g, plan, out) : log_probs<__bf16>(stream, g, plan, out);
}

int dkz_token_log_probs_backward(int type, int rows, int classes, int pitch, const void *logits, float temperature, int given,
                                 const int *tokens, const float *stats, const float *entropy, const float *log_prob_deltas,
                                 const float *entropy_deltas, float beta, void *logits_delta) {
    DKZ_REQUIRE(logits_ok(type, rows, classes, pitch, temperature));
    DKZ_REQUIRE(given >= 0 && given <= kMostGiven);
    if (rows == 0 || classes == 0) return 0;
    const uint64_t m = (uint64_t)rows, n = m * (uint64_t)given, all = logits_bytes(type, rows, classes, pitch);
    DKZ_REQUIRE(logits != nullptr && stats != nullptr && logits_delta != nullptr);
    DKZ_REQUIRE(given == 0 || (tokens != nullptr && log_prob_deltas != nullptr));
    DKZ_REQUIRE(entropy_deltas == nullptr || entropy != nullptr);
    DKZ_REQUIRE(element_aligned(type, logits) && element_aligned(type, logits_delta));
    const bool onto = logits == logits_delta;
    DKZ_REQUIRE(!onto || beta == 0.0f);
    const Span writes[] = {{logits_delta, all}};
    const Span reads[] = {{onto ? nullptr : logits, all}, {tokens, 4 * n}, {stats, 8 * m}, {entropy, 4 * m}, {log_prob_deltas, 4 * n}, {entropy_deltas, 4 * m}};
    DKZ_REQUIRE(disjoint(writes, reads));
    const RowPlan plan = plan_rows(type, rows, classes, ~0ull);
    const Logits g = make_logits(plan, logits, rows, classes, pitch, temperature);
    const Deltas in{tokens, stats, entropy, log_prob_deltas, entropy_deltas, logits_delta, beta, (uint32_t)given};
    const hipStream_t stream = current_stream();
    if (plan.threads == 64) return type == DKZ_F32 ? run_backward<float, 64>(stream, g, plan, in) : run_backward<__bf16, 64>(stream, g, plan, in);
    return type == DKZ_F32 ? run_backward<float, kBlock>(stream, g, plan, in) : run_backward<__bf16, kBlock>(stream, g, plan, in);
}

}  // extern "C"
