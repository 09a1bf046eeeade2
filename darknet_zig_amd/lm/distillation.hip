// distillation.hip -- the divergence from a teacher's top logits, and the delta of
// the logits.
#include "logits.hpp"

namespace dkz {
namespace {

constexpr int kMostEntries = 256;

struct Teacher {
    const int *tokens;
    const float *logits, *row_scales;
    float *loss;
    void *delta;  // null: not wanted
    float scale, temperature;
    uint32_t top;
    // Of rows in several parts: their sums, and the logits of the entries' classes, which the delta may overwrite.
    Sums *part_sums;
    float *entry_logits;  // [rows][kMostEntries]
};

// A row's entries in LDS: their classes, and their probabilities, which are 0 for those that are none.
struct Entries {
    uint32_t token[kMostEntries];
    float p[kMostEntries];
};

// What a group needs to write its part of a row.
template <class T, int THREADS>
struct RowOf {
    static constexpr int kSlots = kMostEntries / THREADS;
    float z[kSlots], log_p[kSlots];  // of this thread's entries: their class's logit, log p
    float mass;                      // the sum that p was divided by: 0 without an entry

    // Reads the entries into `in`: softmax over the entries that are classes.
    __device__ __forceinline__ void read(const Logits &g, const Teacher &t, uint32_t row, Entries &in, float *lds) {
        const T *logits = static_cast<const T *>(g.p) + (uint64_t)row * g.pitch;
        const auto larger = [](float x, float y) { return fmaxf(x, y); };
        const auto sum = [](float x, float y) { return x + y; };
        float v[kSlots], m = neg_inf(), s = 0.0f;
        __syncthreads();  // the last use of `in`
#pragma unroll
        for (int i = 0; i < kSlots; ++i) {
            const uint32_t j = threadIdx.x + i * THREADS;
            const uint64_t at = (uint64_t)row * t.top + j;
            const uint32_t c = j < t.top ? (uint32_t)t.tokens[at] : ~0u;
            v[i] = c < g.classes ? t.logits[at] : neg_inf();
            z[i] = c >= g.classes ? 0.0f : t.entry_logits != nullptr ? t.entry_logits[(uint64_t)row * kMostEntries + j] : load1(logits, c);
            in.token[j] = c < g.classes ? c : ~0u;
            m = fmaxf(m, v[i]);
        }
        m = group_reduce<float, THREADS>(m, lds, larger);
        const float base = m == neg_inf() ? 0.0f : m;
        float e[kSlots];
#pragma unroll
        for (int i = 0; i < kSlots; ++i) {
            v[i] = (v[i] - base) * g.inv;
            e[i] = expf_cw(v[i]);
            s += e[i];
        }
        s = group_reduce<float, THREADS>(s, lds, sum);
        mass = s;
        const float log_s = logf(s);
#pragma unroll
        for (int i = 0; i < kSlots; ++i) {
            in.p[threadIdx.x + i * THREADS] = e[i] == 0.0f ? 0.0f : e[i] / s;
            log_p[i] = v[i] - log_s;
        }
        __syncthreads();
    }

    // The loss, in every thread.
    __device__ __forceinline__ float loss(const Logits &g, const Teacher &t, const Sums &a, float l, const Entries &in, float *lds) const {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kSlots; ++i) {
            const float p = in.p[threadIdx.x + i * THREADS];
            if (p != 0.0f) sum += p * (log_p[i] - log_prob_of(z[i], a.m, l, g.inv));
        }
        return t.temperature * (t.temperature * group_reduce<float, THREADS>(sum, lds, [](float x, float y) { return x + y; }));
    }

    // Writes a part of the delta.
    __device__ __forceinline__ void write(const Logits &g, const Teacher &t, const Part<T> &part, uint32_t row, const Sums &a, float l,
                                          const Entries &in, const Exp<T> &ex) const {
        constexpr int kEach = kTileVectors;
        T *out = static_cast<T *>(t.delta) + (uint64_t)row * g.pitch;
        float factor = t.row_scales != nullptr ? t.scale * t.row_scales[row] : t.scale;
        const bool none = mass == 0.0f || factor == 0.0f || (a.m == neg_inf() && l == neg_inf());
        factor *= t.temperature;
        const auto dense = [&](float z) __attribute__((always_inline)) { return none ? 0.0f : -factor * probability<T>(ex.scaled(z - a.m), l); };
        float fixed[kSlots];
        bool mine[kSlots];
#pragma unroll
        for (int i = 0; i < kSlots; ++i) {
            const uint32_t j = threadIdx.x + i * THREADS, c = in.token[j];
            mine[i] = c != ~0u && part.has(c);
            if (!mine[i]) continue;
            float p = 0.0f;
            for (uint32_t k = 0; k < t.top; ++k) {
                if (in.token[k] != c) continue;
                if (k < j) mine[i] = false;
                p += in.p[k];
            }
            fixed[i] = none ? 0.0f : factor * p + dense(z[i]);
        }
        for (uint32_t v0 = part.v0; v0 < part.v1; v0 += kEach * THREADS) {
            u32x4v raw[kEach];
#pragma unroll
            for (int u = 0; u < kEach; ++u) raw[u] = part.load(v0 + u * THREADS + threadIdx.x);
#pragma unroll
            for (int u = 0; u < kEach; ++u) {
                float d[kVec<T>];
                unpack<T>(raw[u], d);
#pragma unroll
                for (uint32_t i = 0; i < kVec<T>; ++i) d[i] = dense(d[i]);
                part.store_other(out, v0 + u * THREADS + threadIdx.x, d);
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kSlots; ++i)
            if (mine[i]) store1(out, in.token[threadIdx.x + i * THREADS], fixed[i]);
    }
};

template <class T, int THREADS>
__device__ __forceinline__ Sums part_sums(const Part<T> &p, const Exp<T> &ex, Sums *lds) {
    constexpr int kEach = kTileVectors;
    Sums a{neg_inf(), 0.0f, 0.0f};
    for (uint32_t v0 = p.v0; v0 < p.v1; v0 += kEach * THREADS) {
        u32x4v raw[kEach];
#pragma unroll
        for (int u = 0; u < kEach; ++u) raw[u] = p.load(v0 + u * THREADS + threadIdx.x);
        add<T, false>(a, raw, ex);
    }
    return group_reduce<Sums, THREADS>(a, lds, [&](const Sums &x, const Sums &y) { return merge(x, y, ex); });
}

// A group takes a row: its sums, the loss, and the delta in a second pass.
template <class T, int THREADS>
__global__ __launch_bounds__(THREADS) void distillation_kernel(Logits g, Teacher t) {
    __shared__ Sums sums[THREADS / kWave];
    __shared__ float lds[THREADS / kWave];
    __shared__ Entries in;
    const Exp<T> ex(g.inv);
    for (uint32_t row = blockIdx.x; row < g.rows; row += gridDim.x) {
        RowOf<T, THREADS> r;
        r.read(g, t, row, in, lds);
        const Part<T> p(g, row, 0);
        const Sums a = part_sums<T, THREADS>(p, ex, sums);
        const float l = log_sum(a), loss = r.loss(g, t, a, l, in, lds);
        if (threadIdx.x == 0) t.loss[row] = loss;
        if (t.delta != nullptr) r.write(g, t, p, row, a, l, in, ex);
    }
}

// Rows in several parts: the sums of each, then the loss and the delta.
template <class T>
__global__ __launch_bounds__(kBlock) void distillation_sums_kernel(Logits g, Teacher t) {
    __shared__ Sums sums[kBlock / kWave];
    const Exp<T> ex(g.inv);
    const uint32_t row = blockIdx.x / g.parts, part = blockIdx.x - row * g.parts;
    const Sums a = part_sums<T, kBlock>(Part<T>(g, row, part), ex, sums);
    if (threadIdx.x == 0) t.part_sums[blockIdx.x] = a;
    if (part == 0 && threadIdx.x < t.top) {
        const uint32_t c = (uint32_t)t.tokens[(uint64_t)row * t.top + threadIdx.x];
        if (c < g.classes)
            t.entry_logits[(uint64_t)row * kMostEntries + threadIdx.x] = load1(static_cast<const T *>(g.p) + (uint64_t)row * g.pitch, c);
    }
}
template <class T>
__global__ __launch_bounds__(kBlock) void distillation_delta_kernel(Logits g, Teacher t) {
    __shared__ Sums sums[kBlock / kWave];
    __shared__ float lds[kBlock / kWave];
    __shared__ Entries in;
    const Exp<T> ex(g.inv);
    // Without a delta a group a row suffices.
    const uint32_t parts = t.delta != nullptr ? g.parts : 1, row = blockIdx.x / parts, part = blockIdx.x - row * parts;
    RowOf<T, kBlock> r;
    r.read(g, t, row, in, lds);
    Sums a{neg_inf(), 0.0f, 0.0f};
    for (uint32_t p = threadIdx.x; p < g.parts; p += kBlock) a = merge(a, t.part_sums[(uint64_t)row * g.parts + p], ex);
    a = group_reduce<Sums, kBlock>(a, sums, [&](const Sums &x, const Sums &y) { return merge(x, y, ex); });
    const float l = log_sum(a);
    if (part == 0) {
        const float loss = r.loss(g, t, a, l, in, lds);
        if (threadIdx.x == 0) t.loss[row] = loss;
    }
    if (t.delta != nullptr) r.write(g, t, Part<T>(g, row, part), row, a, l, in, ex);
}

uint64_t part_bytes(uint64_t rows, const RowPlan &p) {
    return p.parts == 1 ? 0 : padded(rows * p.parts * sizeof(Sums)) + padded(rows * kMostEntries * 4);
}

template <class T>
int distill(hipStream_t stream, const Logits &g, const RowPlan &plan, const Teacher &t) {
    constexpr const char *kName = "distillation";
    if (plan.parts == 1) {
        const dim3 grid(plan.groups(g.rows));
        if (plan.threads == 64) return launch_on(stream, kName, distillation_kernel<T, 64>, grid, dim3(64), g, t);
        return launch_on(stream, kName, distillation_kernel<T, kBlock>, grid, dim3(kBlock), g, t);
    }
    DKZ_TRY(launch_on(stream, "distillation_sums", distillation_sums_kernel<T>, dim3(g.rows * g.parts), dim3(kBlock), g, t));
    return launch_on(stream, kName, distillation_delta_kernel<T>, dim3(t.delta != nullptr ? g.rows * g.parts : g.rows), dim3(kBlock), g, t);
}

}  // namespace
}  // namespace dkz

using namespace dkz;

extern "C" {

int dkz_distillation_workspace(int type, int rows, int classes, size_t *bytes) {
    DKZ_REQUIRE(bytes != nullptr && logits_ok(type, rows, classes, classes, 1.0f));
    *bytes = (size_t)part_bytes((uint64_t)rows, plan_rows(type, rows, classes));
    return 0;
}

int dkz_distillation(int type, int rows, int classes, int pitch, const void *logits, float temperature, int top,
                     const int *teacher_tokens, const float *teacher_logits, const float *row_scales, float scale, float *loss,
                     void *logits_delta, void *workspace, size_t workspace_bytes) {
    DKZ_REQUIRE(logits_ok(type, rows, classes, pitch, temperature));
    DKZ_REQUIRE(top >= 1 && top <= kMostEntries);
    if (rows == 0) return 0;
    const uint64_t m = (uint64_t)rows, n = m * (uint64_t)top, all = logits_bytes(type, rows, classes, pitch);
    DKZ_REQUIRE(teacher_tokens != nullptr && teacher_logits != nullptr && loss != nullptr && (classes == 0 || logits != nullptr));
    DKZ_REQUIRE(element_aligned(type, logits) && element_aligned(type, logits_delta));
    const RowPlan plan = plan_rows(type, rows, classes);
    const uint64_t need = part_bytes(m, plan);
    DKZ_REQUIRE_WORKSPACE(need);
    const Span writes[] = {{loss, 4 * m}, {logits_delta, all}, {workspace, need}};
    const Span reads[] = {{logits == logits_delta ? nullptr : logits, all}, {teacher_tokens, 4 * n}, {teacher_logits, 4 * n}, {row_scales, 4 * m}};
    DKZ_REQUIRE(disjoint(writes, reads));
    Teacher t{teacher_tokens, teacher_logits, row_scales, loss, logits_delta, scale, temperature, (uint32_t)top, nullptr, nullptr};
    Workspace ws{static_cast<char *>(workspace), need};
    if (plan.parts > 1) {
        t.part_sums = ws.take<Sums>(m * plan.parts);
        t.entry_logits = ws.take<float>(m * kMostEntries);
    }
    const Logits g = make_logits(plan, logits, rows, classes, pitch, temperature);
    const hipStream_t stream = current_stream();
    return type == DKZ_F32 ? distill<float>(stream, g, plan, t) : distill<__bf16>(stream, g, plan, t);
}

}  // extern "C"
