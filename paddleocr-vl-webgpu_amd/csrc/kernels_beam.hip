// Beam search's selection: the best continuations over beams and vocabulary.
//
// A beam b with score s_b continues with token t at s_b + x_t - lse, lse =
// log sum exp(x) over its row of logits.  One pass over the logits: a workgroup
// takes a segment of a row and leaves its largest logit, its sum of exponentials
// and its best candidates; a second launch joins the segments of a row and, as
// the last row of a batch entry to finish, the rows.
//
// Order.  Within a row candidates are ordered by logit, then by token: one
// 64-bit key, (the logit's bits, made monotone) * 2^32 + (2^32 - 1 - token), so no
// two are equal and the larger is the better.  Across rows by score, in 64 bits
// (scores of two beams may lie closer than f32 tells apart, and the order of
// what is returned must not depend on it), then by beam, then by key.
//
// The best n of many without sorting them: with the values dealt to threads, the
// n-th largest of the threads' own largest is a bound that at least n values
// reach, and only values of n threads can reach it, so a short list remains,
// whose ranks are counted.

#include <hip/hip_runtime.h>

#include <cstdint>

#include "pvlc_device.hpp"
#include "pvlc_internal.hpp"

namespace pvlc {
namespace {

typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

constexpr float kLargestFloat = 3.402823466e38f;

// NaN counts as masked (-inf), +inf as the largest finite value.
__device__ inline float clean(float x) { return x != x ? -INFINITY : fminf(x, kLargestFloat); }

__device__ inline uint64_t key_of(float x, uint32_t token) {
    const int32_t bits = __float_as_int(x);
    const uint32_t order = static_cast<uint32_t>(bits ^ ((bits >> 31) & 0x7FFFFFFF)) ^ 0x80000000u;
    return static_cast<uint64_t>(order) << 32 | (0xFFFFFFFFu - token);
}
__device__ inline float logit_of(uint64_t key) {
    const int32_t order = static_cast<int32_t>(static_cast<uint32_t>(key >> 32) ^ 0x80000000u);
    return __int_as_float(order ^ ((order >> 31) & 0x7FFFFFFF));
}
__device__ inline uint32_t token_of(uint64_t key) { return 0xFFFFFFFFu - static_cast<uint32_t>(key); }
constexpr uint64_t kNoKey = 0;  // below every logit's key (a NaN's, which none has)

// exp(x) for x <= 0.  The product with log2(e) in two parts: the rounded
// constant alone shifts a term by 1.3e-8 of its exponent.
__device__ inline float exp_of(float x) {
    const float y = fmaxf(x, -200.f);  // 0 below, -inf among it
    const float hi = y * 1.44269502f;
    return __builtin_amdgcn_exp2f(hi + (__builtin_fmaf(y, 1.44269502f, -hi) + y * 1.92596299e-8f));
}

// A beam goes on if its score is above -inf (not NaN), a row of logits is read
// if the beam is also not finished.
__device__ inline bool row_finished(const BeamSelect &b, uint32_t row) { return b.finished != nullptr && b.finished[row] != 0; }
__device__ inline bool row_alive(const BeamSelect &b, uint32_t row) { return b.scores[row] > -INFINITY; }

// Order of a row's candidates: the key; of a batch entry's: score, then the lower
// number (beam, and rank in its row).
struct Scored {
    double score;  // -inf: none
    uint32_t number;
    uint32_t pad;
};
__device__ inline bool better(uint64_t a, uint64_t b) { return a > b; }
__device__ inline bool better(const Scored &a, const Scored &b) { return a.score > b.score || (a.score == b.score && a.number < b.number); }
__device__ inline bool is_any(uint64_t a) { return a != kNoKey; }
__device__ inline bool is_any(const Scored &a) { return a.score > -INFINITY; }

// LDS of best_of: the threads' own largest, the short list, the bound.
template <class Item, int kEach>
struct BestLds {
    Item most[kBeamThreads];
    Item list[kBeamMaxBest * kEach];
    Item bound;
    uint32_t count;
};

// The `best` best of the workgroup's items, kEach a thread, in order: put(rank,
// item) for each of them, as many as there are.  No two items are equal.  Every
// thread calls it; what put writes to LDS is seen after the next barrier.
template <int kEach, class Item, class Put>
__device__ inline void best_of(const Item (&item)[kEach], const Item &none, uint32_t best, BestLds<Item, kEach> &lds, Put put) {
    const uint32_t i = threadIdx.x;
    Item own = none;
#pragma unroll
    for (int e = 0; e < kEach; ++e)
        if (better(item[e], own)) own = item[e];
    lds.most[i] = own;
    if (i == 0) {
        lds.bound = none;
        lds.count = 0;
    }
    __syncthreads();
    uint32_t above = 0;
#pragma unroll 8
    for (uint32_t j = 0; j < kBeamThreads; ++j) above += better(lds.most[j], own);
    const bool in = is_any(own) && above < best;
    if (in && above == best - 1) lds.bound = own;  // one thread at most; without it all items of fewer than `best` threads are listed
    __syncthreads();
    if (in) {
        const Item bound = lds.bound;
#pragma unroll
        for (int e = 0; e < kEach; ++e)
            if (is_any(item[e]) && !better(bound, item[e])) lds.list[atomicAdd(&lds.count, 1u)] = item[e];
    }
    __syncthreads();
    const uint32_t n = lds.count;
    for (uint32_t c = i; c < n; c += kBeamThreads) {
        const Item mine = lds.list[c];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < n; ++j) rank += better(lds.list[j], mine);
        if (rank < best) put(rank, mine);
    }
}

template <class T, class Op>
__device__ inline T workgroup_reduce(T v, T *sm, Op op) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o));
    __syncthreads();  // sm's readers before are done
    if (lane == 0) sm[threadIdx.x >> 6] = v;
    __syncthreads();
    T r = sm[0];
#pragma unroll
    for (uint32_t w = 1; w < kBeamThreads / 64; ++w) r = op(r, sm[w]);
    return r;
}
__device__ inline float larger(float a, float b) { return fmaxf(a, b); }
__device__ inline double plus(double a, double b) { return a + b; }

// Grid (segment, row).
__global__ __launch_bounds__(kBeamThreads) void beam_segment_kernel(BeamSelect b) {
    __shared__ BestLds<uint64_t, kBeamEach> lds;
    __shared__ float sm_f[kBeamThreads / 64];
    __shared__ double sm_d[kBeamThreads / 64];
    const uint32_t segment = blockIdx.x, row = blockIdx.y, i = threadIdx.x;
    if (!row_alive(b, row) || row_finished(b, row)) return;  // uniform; the row's join reads nothing then
    const float *x = b.logits + static_cast<uint64_t>(row) * b.row_stride;
    const uint32_t first = segment * kBeamSegment;
    float v[kBeamEach];
#pragma unroll
    for (uint32_t c = 0; c < kBeamEach / 4; ++c) {
        const uint32_t at = first + (c * kBeamThreads + i) * 4;
        if (b.vocab - first >= kBeamSegment) {  // uniform
            const f32x4_any q = __builtin_nontemporal_load(reinterpret_cast<const f32x4_any *>(x + at));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[c * 4 + e] = q[e];
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) v[c * 4 + e] = at + e < b.vocab ? x[at + e] : -INFINITY;
        }
    }
    float most = -INFINITY;
    uint64_t key[kBeamEach];
#pragma unroll
    for (uint32_t e = 0; e < kBeamEach; ++e) {
        v[e] = clean(v[e]);
        most = fmaxf(most, v[e]);
        key[e] = v[e] > -INFINITY ? key_of(v[e], first + ((e >> 2) * kBeamThreads + i) * 4 + (e & 3)) : kNoKey;
    }
    most = workgroup_reduce(most, sm_f, larger);
    float sum = 0.f;
#pragma unroll
    for (uint32_t e = 0; e < kBeamEach; ++e) sum += exp_of(v[e] - most);  // (NaN where all are masked: not used)
    const double total = workgroup_reduce(static_cast<double>(sum), sm_d, plus);
    const size_t part = static_cast<size_t>(row) * b.segments + segment;
    if (i == 0) {
        b.largest[part] = most;
        b.sums[part] = most > -INFINITY ? total : 0.0;
    }
    uint64_t *out = b.keys + part * b.best;
    best_of(key, kNoKey, b.best, lds, [&](uint32_t rank, uint64_t k) { out[rank] = k; });
    for (uint32_t k = min(lds.count, b.best) + i; k < b.best; k += kBeamThreads) out[k] = kNoKey;
}

__device__ inline void store_agent(uint64_t *p, uint64_t v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ inline uint64_t load_agent(const uint64_t *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// A workgroup joins the segments of a row; the last row of a batch entry joins
// its rows (relaxed agent-scope stores, their acknowledgement, a counter, and
// agent-scope loads, as the split decode's partitions).
__global__ __launch_bounds__(kBeamThreads) void beam_join_kernel(BeamSelect b) {
    constexpr int kEach = kBeamEach + 1;  // a round's items, and one of the best so far
    __shared__ union {
        BestLds<uint64_t, kEach> keys;
        BestLds<Scored, kEach> scored;
    } lds;
    __shared__ uint64_t run[kBeamMaxBest];
    __shared__ Scored run_scored[kBeamMaxBest];
    __shared__ float sm_f[kBeamThreads / 64];
    __shared__ double sm_d[kBeamThreads / 64];
    __shared__ int sm_last;
    const uint32_t row = blockIdx.x, i = threadIdx.x, entry = row / b.beams;
    const float start = b.scores[row];
    const bool finished = row_finished(b, row);
    for (uint32_t k = i; k < b.best; k += kBeamThreads) run[k] = kNoKey;
    __syncthreads();
    double lse = 0.0;
    if (start > -INFINITY && finished) {
        if (i == 0) run[0] = 0x8000000000000000ull | (0xFFFFFFFFu - static_cast<uint32_t>(b.end_token));
    } else if (start > -INFINITY) {
        const size_t part = static_cast<size_t>(row) * b.segments;
        float most = -INFINITY;
        for (uint32_t s = i; s < b.segments; s += kBeamThreads) most = fmaxf(most, b.largest[part + s]);
        most = workgroup_reduce(most, sm_f, larger);
        double sum = 0.0;
        if (most > -INFINITY)  // uniform
            for (uint32_t s = i; s < b.segments; s += kBeamThreads) sum += b.sums[part + s] * exp(static_cast<double>(b.largest[part + s]) - most);
        sum = workgroup_reduce(sum, sm_d, plus);
        lse = most + log(sum);
        if (most > -INFINITY) {
            const uint64_t *keys = b.keys + part * b.best;
            const uint64_t items = static_cast<uint64_t>(b.segments) * b.best;
            for (uint64_t at = 0; at < items; at += kBeamSegment) {
                uint64_t key[kEach];
#pragma unroll
                for (uint32_t e = 0; e < kBeamEach; ++e) {
                    const uint64_t k = at + e * kBeamThreads + i;
                    key[e] = k < items ? keys[k] : kNoKey;
                }
                key[kBeamEach] = i < b.best ? run[i] : kNoKey;
                best_of(key, kNoKey, b.best, lds.keys, [&](uint32_t rank, uint64_t k) { run[rank] = k; });
                __syncthreads();
            }
        }
    }
    __syncthreads();
    // (thread i holds rank i of the row)
    auto score_of = [&](uint64_t key) {
        return finished ? static_cast<double>(start) : start + (static_cast<double>(logit_of(key)) - lse);
    };
    if (b.beams > 1) {
        if (i < b.best) {
            const size_t at = static_cast<size_t>(row) * b.best + i;
            const uint64_t key = run[i];
            store_agent(b.row_keys + at, key);
            store_agent(reinterpret_cast<uint64_t *>(b.row_scores) + at,
                        static_cast<uint64_t>(__double_as_longlong(key != kNoKey ? score_of(key) : -INFINITY)));
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (i == 0) sm_last = __hip_atomic_fetch_add(b.arrived + entry, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == b.beams - 1;
        __syncthreads();
        if (!sm_last) return;
        if (i == 0) __hip_atomic_store(b.arrived + entry, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    const Scored none{-INFINITY, UINT32_MAX, 0};
    for (uint32_t k = i; k < b.best; k += kBeamThreads) run_scored[k] = none;
    __syncthreads();
    const size_t rows_at = static_cast<size_t>(entry) * b.beams * b.best;
    if (b.beams > 1) {
        const uint32_t items = b.beams * b.best;
        for (uint32_t at = 0; at < items; at += kBeamSegment) {
            Scored s[kEach];
#pragma unroll
            for (uint32_t e = 0; e < kBeamEach; ++e) {
                const uint32_t k = at + e * kBeamThreads + i;
                s[e] = none;
                if (k < items)
                    s[e] = Scored{__longlong_as_double(static_cast<long long>(load_agent(reinterpret_cast<const uint64_t *>(b.row_scores) + rows_at + k))), k, 0};
            }
            s[kBeamEach] = i < b.best ? run_scored[i] : none;
            best_of(s, none, b.best, lds.scored, [&](uint32_t rank, const Scored &c) { run_scored[rank] = c; });
            __syncthreads();
        }
    } else if (i < b.best && run[i] != kNoKey) {
        run_scored[i] = Scored{score_of(run[i]), i, 0};
    }
    __syncthreads();
    if (i >= b.best) return;
    const Scored c = run_scored[i];
    const bool any = c.score > -INFINITY;
    const uint32_t parent = entry * b.beams + c.number / b.best;
    int32_t token = -1;
    if (any) token = static_cast<int32_t>(token_of(b.beams > 1 ? load_agent(b.row_keys + rows_at + c.number) : run[c.number]));
    const size_t o = static_cast<size_t>(entry) * b.best + i;
    b.next_scores[o] = any ? static_cast<float>(c.score) : -INFINITY;
    b.parents[o] = any ? static_cast<int32_t>(parent) : -1;
    b.tokens[o] = token;
    if (b.next_finished) b.next_finished[o] = any && (token == b.end_token || row_finished(b, parent));
}

}  // namespace

int launch_beam_select(const BeamSelect &b, void *stream) {
    const hipStream_t st = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(beam_segment_kernel, dim3(b.segments, b.batch * b.beams), dim3(kBeamThreads), 0, st, b);
    hipLaunchKernelGGL(beam_join_kernel, dim3(b.batch * b.beams), dim3(kBeamThreads), 0, st, b);
    return static_cast<int>(hipGetLastError());
}

}  // namespace pvlc
