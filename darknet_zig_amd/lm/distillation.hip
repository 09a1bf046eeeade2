// distillation.hip -- the divergence from a teacher's top logits, and the delta of
// the logits.
#include "logits.hpp"

namespace dkz {
namespace {

constexpr int kMostEntries = 256;
constexpr uint64_t kMostParts = 64;  // of a row: each one's group joins all their sums
constexpr uint32_t kMostPartGroups = 1u << 20;  // of a launch

struct Teacher {
    const int *tokens;
    const float *logits, *row_scales;
    float *loss;
    void *delta;  // null: not wanted
    float scale, temperature;
    uint32_t top;
    // Of rows in parts: their sums, and the logits of the entries' classes, which the delta may overwrite.
    Sums *part_sums;
    float *entry_logits;  // [rows][kMostEntries]
};

// A row's entries in LDS, for all of its group: their classes (~0: none) and probabilities, which are 0 for those that are
// none, and the sum that those were divided by: 0 without an entry.
struct __align__(16) Entries {
    uint32_t token[kMostEntries];
    float p[kMostEntries], log_p[kMostEntries], z[kMostEntries];  // log_p, z: for the loss, and their class's logit
    float mass;
};

// What a group does with a row's entries. Its first wave has them, one a lane and then the next 64: loops over them are kept
// as loops, since all of this stands beside a row's logits in registers.
template <class T>
struct RowOf {
    const Logits &g;
    const Teacher &t;
    Entries &in;
    uint32_t row;
    const T *logits;
    uint32_t c;  // of the lane's first entry: its class, logit, and its class's logit here
    float v, z;

    __device__ __forceinline__ RowOf(const Logits &g, const Teacher &t, Entries &in, uint32_t row)
        : g(g), t(t), in(in), row(row), logits(static_cast<const T *>(g.p) + (uint64_t)row * g.pitch) {}

    __device__ __forceinline__ void entry(uint32_t j) {
        const uint64_t at = (uint64_t)row * t.top + j;
        c = ~0u;
        v = neg_inf();
        if (j < t.top) {
            c = (uint32_t)t.tokens[at];
            v = t.logits[at];
        }
    }
    __device__ __forceinline__ void class_logit(uint32_t j) {
        z = 0.0f;
        if (c >= g.classes) {
            c = ~0u;
            v = neg_inf();
        } else {
            z = t.entry_logits != nullptr ? t.entry_logits[(uint64_t)row * kMostEntries + j] : load1(logits, c);
        }
    }
    // The first entries' loads, apart so that others are issued between them.
    __device__ __forceinline__ void begin() { entry(threadIdx.x); }
    __device__ __forceinline__ void gather() { class_logit(threadIdx.x); }
    // Softmax over the entries that are classes. A lane looks at its own entries in LDS alone: no barrier. The first entries' z is
    // on its way and not looked at.
    __device__ __forceinline__ void finish() {
        const float first_z = z;
        float m = v, s = 0.0f;
        in.token[threadIdx.x] = c;
        in.log_p[threadIdx.x] = v;
#pragma unroll 1
        for (uint32_t j = threadIdx.x + kWave; j - threadIdx.x < t.top; j += kWave) {
            entry(j);
            class_logit(j);
            in.token[j] = c;
            in.log_p[j] = v;
            in.z[j] = z;
            m = fmaxf(m, v);
        }
        z = first_z;
        m = lanes_reduce<kWave>(m, [](float x, float y) { return fmaxf(x, y); });
        const float base = m == neg_inf() ? 0.0f : m;
#pragma unroll 1
        for (uint32_t j = threadIdx.x; j - threadIdx.x < t.top; j += kWave) {
            const float y = (in.log_p[j] - base) * g.inv, e = expf_cw(y);
            in.log_p[j] = y;
            in.p[j] = e;
            s += e;
        }
        s = lanes_reduce<kWave>(s, [](float x, float y) { return x + y; });
        const float log_s = logf(s), over = 1.0f / s;
#pragma unroll 1
        for (uint32_t j = threadIdx.x; j - threadIdx.x < t.top; j += kWave) {
            // NaN: a NaN or infinity among them leaves no entry a probability.
            in.p[j] = in.p[j] == 0.0f && (s == s || in.token[j] == ~0u) ? 0.0f : in.p[j] * over;
            in.log_p[j] -= log_s;
        }
        if (threadIdx.x == 0) in.mass = s;
    }
    __device__ __forceinline__ void read() {
        begin();
        gather();
        finish();
    }

    // The loss, by the first wave. temperature * (log p - log q) is temperature * (log p + l) - (z - m), which stays finite where
    // a class is masked by the type's lowest value and the temperature is below 1.
    __device__ __forceinline__ void loss(const Sums &a, float l, bool store = true) const {
        const bool left = a.m != neg_inf() || l != neg_inf();  // a class
        float sum = 0.0f;
        in.z[threadIdx.x] = z;
#pragma unroll 1
        for (uint32_t j = threadIdx.x; j < t.top; j += kWave)
            if (in.p[j] != 0.0f) sum += in.p[j] * (left ? t.temperature * (in.log_p[j] + l) - (in.z[j] - a.m) : -neg_inf());
        sum = lanes_reduce<kWave>(sum, [](float x, float y) { return x + y; });
        if (threadIdx.x == 0 && store) t.loss[row] = t.temperature * sum;
    }

    // Writes a part of the delta. vectors(f) calls f(v, logits of vector v) for this thread's vectors of the part.
    template <int THREADS, class F>
    __device__ __forceinline__ void write(const Part<T> &part, const Sums &a, float l, const Exp<T> &ex, F vectors) const {
        T *out = static_cast<T *>(t.delta) + (uint64_t)row * g.pitch;
        float factor = t.row_scales != nullptr ? t.scale * t.row_scales[row] : t.scale;
        const bool none = in.mass == 0.0f || factor == 0.0f || (a.m == neg_inf() && l == neg_inf());
        factor *= t.temperature;
        const auto dense = [&](float z) __attribute__((always_inline)) { return none ? 0.0f : -factor * probability<T>(z - a.m, l, ex); };
        vectors([&](uint32_t v, const u32x4v &raw) __attribute__((always_inline)) {
            float d[kVec<T>];
            unpack<T>(raw, d);
#pragma unroll
            for (uint32_t i = 0; i < kVec<T>; ++i) d[i] = dense(d[i]);
            part.store_other(out, v, d);
        });
        if (const uint32_t c = part.edge(); c != ~0u) store1(out, c, dense(load1(logits, c)));
        // The entries' classes are written a second time, when the others have been, by the thread that has a class's first entry.
        __syncthreads();
#pragma unroll 1
        for (uint32_t j = threadIdx.x; j < t.top; j += THREADS) {
            const uint32_t c = in.token[j];
            if (c == ~0u || !part.has(c)) continue;
            const Claim own = claim(in.token, in.p, t.top, j, c);
            if (own.first) store1(out, c, none ? 0.0f : factor * own.sum + dense(in.z[j]));
        }
    }
    // The same, from logits that are read again.
    template <int THREADS>
    __device__ __forceinline__ void write_again(const Part<T> &part, const Sums &a, float l, const Exp<T> &ex) const {
        write<THREADS>(part, a, l, ex, [&](auto f) __attribute__((always_inline)) {
            constexpr int kEach = kTileVectors;
            for (uint32_t v0 = part.v0 + threadIdx.x; v0 < part.v1; v0 += kEach * THREADS) {
                u32x4v raw[kEach];
                part.load(v0, THREADS, raw);
#pragma unroll
                for (int u = 0; u < kEach; ++u)
                    if (v0 + u * THREADS < part.v1) f(v0 + u * THREADS, raw[u]);
            }
        });
    }
};

template <class T, int THREADS>
__device__ __forceinline__ Sums part_sums(const T *logits, const Part<T> &p, const Exp<T> &ex, Sums *lds) {
    constexpr int kEach = kTileVectors;
    Sums a{neg_inf(), 0.0f, 0.0f};
    for (uint32_t v0 = p.v0; v0 < p.v1; v0 += kEach * THREADS) {
        u32x4v raw[kEach];
        p.load(v0 + threadIdx.x, THREADS, raw);
        float largest[kEach];
        add_until<T, false>(a, raw, largest, v0 + threadIdx.x, THREADS, p.v1, ex);
    }
    const uint32_t edge = p.edge();
    add_one(a, edge != ~0u ? load1(logits, edge) : neg_inf(), ex);
    return group_reduce<Sums, THREADS>(a, lds, [&](const Sums &x, const Sums &y) { return merge(x, y, ex); });
}

// A group takes a row, which it holds in registers, U vectors a thread, from the sums to the delta: every logit is
// read once.
template <class T, int THREADS, int U>
__global__ __launch_bounds__(THREADS, U == 16 ? 4 : U == 8 ? 6 : 8) void distillation_held_kernel(Logits g, Teacher t) {
    __shared__ Sums sums[THREADS / kWave];
    __shared__ Entries in;
    const Exp<T> ex(g.inv);
    const bool first = threadIdx.x < kWave;
    for (uint32_t row = blockIdx.x; row < g.rows; row += gridDim.x) {
        const Part<T> p(g, row, 0);
        RowOf<T> r(g, t, in, row);
        if (first) r.begin();
        u32x4v raw[U];
        p.load(p.v0 + threadIdx.x, THREADS, raw);
        const uint32_t edge = p.edge();
        const float at_edge = edge != ~0u ? load1(r.logits, edge) : neg_inf();
        if (row != blockIdx.x) __syncthreads();  // the last row's use of `in`
        if (first) {
            r.gather();
            r.finish();
        }
        Sums a = sums_of<T>(raw, ex);
        add_one(a, at_edge, ex);
        a = group_reduce<Sums, THREADS>(a, sums, [&](const Sums &x, const Sums &y) { return merge(x, y, ex); });
        if constexpr (THREADS == kWave) __syncthreads();  // else the sums' have done it
        const float l = log_sum(a);
        if (first) r.loss(a, l);
        if (t.delta != nullptr)
            r.template write<THREADS>(p, a, l, ex, [&](auto f) __attribute__((always_inline)) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const uint32_t v = p.v0 + u * THREADS + threadIdx.x;
                    if (v < p.v1) f(v, raw[u]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            });
    }
}

// Rows in parts: the sums of each, then the loss and the delta.
template <class T>
__global__ __launch_bounds__(kBlock) void distillation_sums_kernel(Logits g, Teacher t) {
    __shared__ Sums sums[kBlock / kWave];
    const Exp<T> ex(g.inv);
    const uint32_t row = blockIdx.x / g.parts, part = blockIdx.x - row * g.parts;
    const T *logits = static_cast<const T *>(g.p) + (uint64_t)row * g.pitch;
    const Sums a = part_sums<T, kBlock>(logits, Part<T>(g, row, part), ex, sums);
    if (threadIdx.x == 0) t.part_sums[blockIdx.x] = a;
    if (part == 0 && threadIdx.x < t.top) {
        const uint32_t c = (uint32_t)t.tokens[(uint64_t)row * t.top + threadIdx.x];
        if (c < g.classes) t.entry_logits[(uint64_t)row * kMostEntries + threadIdx.x] = load1(logits, c);
    }
}
template <class T>
__global__ __launch_bounds__(kBlock) void distillation_delta_kernel(Logits g, Teacher t) {
    __shared__ Sums sums[kBlock / kWave];
    __shared__ Entries in;
    const Exp<T> ex(g.inv);
    // Without a delta a group a row suffices.
    const uint32_t parts = t.delta != nullptr ? g.parts : 1, row = blockIdx.x / parts, part = blockIdx.x - row * parts;
    RowOf<T> r(g, t, in, row);
    if (threadIdx.x < kWave) r.read();
    Sums a{neg_inf(), 0.0f, 0.0f};
    for (uint32_t p = threadIdx.x; p < g.parts; p += kBlock) a = merge(a, t.part_sums[(uint64_t)row * g.parts + p], ex);
    a = group_reduce<Sums, kBlock>(a, sums, [&](const Sums &x, const Sums &y) { return merge(x, y, ex); });
    const float l = log_sum(a);
    if (threadIdx.x < kWave) r.loss(a, l, part == 0);
    if (t.delta != nullptr) r.template write_again<kBlock>(Part<T>(g, row, part), a, l, ex);
}

// How rows are taken: held by groups of `threads` with `vectors` a thread, or (threads 0) in parts.
struct DistillPlan {
    uint32_t threads, vectors;
    RowPlan rows;
    uint64_t bytes(uint64_t n) const { return threads != 0 ? 0 : padded(n * rows.parts * sizeof(Sums)) + padded(n * kMostEntries * 4); }
};
constexpr uint64_t kFewRows = 64;
DistillPlan plan_distillation(int type, uint64_t rows, uint64_t classes) {
    const uint64_t vectors = classes / (type == DKZ_F32 ? 4 : 8);  // whole ones at most
    // 4096 rows of 65536 bf16 classes 216 us with 512 threads and 16 vectors, 249 with 1024 and 8, 348 with 1024 and 16; of 32768
    // classes 117 with 512 and 8, 124 with 256 and 16, 140 with 1024 and 4.
    constexpr uint32_t kHeld[][2] = {{64, 4}, {256, 4}, {256, 8}, {512, 8}, {512, 16}, {1024, 16}};
    for (const auto &h : kHeld) {
        // Few long rows leave the chip empty: two launches of several groups a row (65536 classes in bf16: 1 row 11.0 us, 13.3
        // held; 64 rows 16.3 and 17.1; 128 rows 19.4 and 18.0. 131072: 1 row 11.0 and 20.7, 64 rows 19.0 and 25.0. 32768: 1 row
        // 10.6 and 9.5). One limit for all lengths, 65536 classes': for 131072 it comes early (64 rows 17.9 in parts, 65 rows 21.8 held).
        if (rows <= kFewRows && h[0] * h[1] > 4096) break;
        if (vectors <= h[0] * h[1]) return {h[0], h[1], {0, 1, h[0] * h[1]}};
    }
    return {0, 0, plan_rows(type, rows, classes, kMostParts * rows)};
}
// The most that any number of rows up to `rows` takes: those in parts take more the more they are.
uint64_t most_bytes(int type, uint64_t rows, uint64_t classes) {
    const uint64_t few = std::min(rows, kFewRows);
    return std::max(plan_distillation(type, rows, classes).bytes(rows), plan_distillation(type, few, classes).bytes(few));
}

// Rows [first, first + n) of the logits, and what belongs to those from `first` on.
template <class T>
Logits rows_of(Logits g, uint64_t first, uint32_t n) {
    g.p = static_cast<const T *>(g.p) + first * g.pitch;
    g.rows = n;
    return g;
}
template <class T>
Teacher rows_of(Teacher t, const Logits &g, uint64_t first) {
    t.tokens += first * t.top;
    t.logits += first * t.top;
    t.row_scales = t.row_scales != nullptr ? t.row_scales + first : nullptr;
    t.loss += first;
    t.delta = t.delta != nullptr ? static_cast<T *>(t.delta) + first * g.pitch : nullptr;
    t.part_sums += first * g.parts;
    t.entry_logits += first * kMostEntries;
    return t;
}

template <class T>
int distill(hipStream_t stream, const Logits &g, const DistillPlan &plan, const Teacher &t) {
    constexpr const char *kName = "distillation";
    const dim3 grid(std::min(g.rows, 1u << 20)), block(plan.threads);
    if (plan.threads == 64) return launch_on(stream, kName, distillation_held_kernel<T, 64, 4>, grid, block, g, t);
    if (plan.threads == 256 && plan.vectors == 4) return launch_on(stream, kName, distillation_held_kernel<T, 256, 4>, grid, block, g, t);
    if (plan.threads == 256) return launch_on(stream, kName, distillation_held_kernel<T, 256, 8>, grid, block, g, t);
    if (plan.threads == 512 && plan.vectors == 8) return launch_on(stream, kName, distillation_held_kernel<T, 512, 8>, grid, block, g, t);
    if (plan.threads == 512) return launch_on(stream, kName, distillation_held_kernel<T, 512, 16>, grid, block, g, t);
    if (plan.threads == 1024) return launch_on(stream, kName, distillation_held_kernel<T, 1024, 16>, grid, block, g, t);
    // A group a part: more of them than a launch counts threads for where the logits are a large part of the memory, so that those
    // take several launches. (One whose groups go round the parts: 64 rows of 65536 classes 13.5 -> 14.3 us, 2000 of 150000 343 -> 357.)
    const uint32_t most = std::max(kMostPartGroups / g.parts, 1u);
    for (uint32_t first = 0; first < g.rows; first += most) {
        const Logits some = rows_of<T>(g, first, std::min(g.rows - first, most));
        const Teacher its = rows_of<T>(t, g, first);
        DKZ_TRY(launch_on(stream, "distillation_sums", distillation_sums_kernel<T>, dim3(some.rows * g.parts), dim3(kBlock), some, its));
        const dim3 groups(t.delta != nullptr ? some.rows * g.parts : some.rows);
        DKZ_TRY(launch_on(stream, kName, distillation_delta_kernel<T>, groups, dim3(kBlock), some, its));
    }
    return 0;
}

}  // namespace
}  // namespace dkz

using namespace dkz;

extern "C" {

int dkz_distillation_workspace(int type, int rows, int classes, size_t *bytes) {
    DKZ_REQUIRE(bytes != nullptr && logits_ok(type, rows, classes, classes, 1.0f));
    *bytes = (size_t)most_bytes(type, (uint64_t)rows, (uint64_t)classes);
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
    const DistillPlan plan = plan_distillation(type, rows, classes);
    const uint64_t need = plan.bytes(m);
    DKZ_REQUIRE_WORKSPACE(need);
    const Span writes[] = {{loss, 4 * m}, {logits_delta, all}, {workspace, need}};
    const Span reads[] = {{logits == logits_delta ? nullptr : logits, all}, {teacher_tokens, 4 * n}, {teacher_logits, 4 * n}, {row_scales, 4 * m}};
    DKZ_REQUIRE(disjoint(writes, reads));
    Teacher t{teacher_tokens, teacher_logits, row_scales, loss, logits_delta, scale, temperature, (uint32_t)top, nullptr, nullptr};
    Workspace ws{static_cast<char *>(workspace), need};
    if (need != 0) {
        t.part_sums = ws.take<Sums>(m * plan.rows.parts);
        t.entry_logits = ws.take<float>(m * kMostEntries);
    }
    const Logits g = make_logits(plan.rows, logits, rows, classes, pitch, temperature);
    const hipStream_t stream = current_stream();
    return type == DKZ_F32 ? distill<float>(stream, g, plan, t) : distill<__bf16>(stream, g, plan, t);
}

}  // extern "C"
