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
// two are equal and the larger is the better.  Across rows by score, in 64 bits:
// scores of two beams may lie closer than f32 tells apart, and the order of what
// is returned must not depend on it (nor on the batch: a row's score is the same
// in any, though its sum's terms are f32).  Again one key: the score's bits, made
// monotone, with the lowest 13 given to the candidate's number (beam, then rank
// in its row), so that scores equal to 2^-39 go by beam and rank.
//
// The best n of many without sorting them: with the values dealt to groups of
// threads, the n-th largest of the groups' own largest is a bound that at least n
// values reach and few others, so a short list remains, whose ranks are counted.
//
// Measured: four rows of 103424 logits, four candidates: segments 4.9-5.1 us, join
// 5.8-6.0 (1.65 MB; both are a launch and a chain of rounds through memory and
// barriers: of the join's, by time stamps, loads 0.7, selection 1.6, the hand-off
// 0.8, loads and selection among the rows 0.9, outputs 0.5).  128 rows, a fifth of
// them finished, sixteen candidates of eight rows each: segments 11.4-12.4 us (42 MB,
// 3.4-3.7 TB/s: a row's loads, exponentials and selection follow one another in
// each workgroup, and little more than one round of workgroups covers the other's
// waits), join 6.9-7.7.  One launch for both, the last segment of a row joining it,
// took 11.7 and 32.6 us a call against 9.9 and 22.9: each segment then waits for
// its stores and an atomic, and the join's registers are every segment's.

#include <hip/hip_runtime.h>

#include <cstdint>

#include "pvlc_device.hpp"
#include "pvlc_internal.hpp"

namespace pvlc {
namespace {

typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

// Logits above 2^127 (and +inf) count as 2^127 and those below -2^127 as masked,
// like -inf and NaN: so masks of the type's lowest value are masks.
constexpr float kMostLogit = 1.7014118346046923e38f;
__device__ inline float clean(float x) { return x != x ? -INFINITY : fminf(x, kMostLogit); }

// A logit's bits as a whole number in its order (-0 below +0), and back.
__device__ inline int32_t order_of(float x) {
    const int32_t bits = __float_as_int(x);
    return bits ^ ((bits >> 31) & 0x7FFFFFFF);
}
__device__ inline float value_of(int32_t order) { return __int_as_float(order ^ ((order >> 31) & 0x7FFFFFFF)); }
constexpr int32_t kLeastOrder = static_cast<int32_t>(0xFF000000u ^ 0x7FFFFFFFu);  // of -2^127

__device__ inline uint64_t key_of(int32_t order, uint32_t token) {
    return static_cast<uint64_t>(static_cast<uint32_t>(order) ^ 0x80000000u) << 32 | (0xFFFFFFFFu - token);
}
__device__ inline int32_t order_in(uint64_t key) { return static_cast<int32_t>(static_cast<uint32_t>(key >> 32) ^ 0x80000000u); }
__device__ inline uint32_t token_in(uint64_t key) { return 0xFFFFFFFFu - static_cast<uint32_t>(key); }
constexpr uint64_t kNoKey = 0;  // below every candidate's key

// A score's key, and the score to 2^-39 and the candidate's number back.
constexpr uint32_t kNumbers = 8192;
static_assert(kBeamMaxBeams * kBeamMaxBest <= kNumbers, "a candidate's number fits a score's key");
__device__ inline uint64_t score_key(double score, uint32_t number) {
    const int64_t bits = __double_as_longlong(score);
    const uint64_t order = static_cast<uint64_t>(bits ^ ((bits >> 63) & 0x7FFFFFFFFFFFFFFFll)) ^ 0x8000000000000000ull;
    return (order & ~static_cast<uint64_t>(kNumbers - 1)) | (kNumbers - 1 - number);
}
__device__ inline uint32_t number_in(uint64_t key) { return kNumbers - 1 - (static_cast<uint32_t>(key) & (kNumbers - 1)); }

// exp(x - reference), x <= reference.  log2(e) in two parts: the rounded constant
// alone shifts a term by 1.3e-8 of its exponent.
__device__ inline float exp_term(float x, float reference) {
    const float d = x - reference;
    return __builtin_amdgcn_exp2f(__builtin_fmaf(d, 1.44269502f, d * 1.92596299e-8f));
}

// A beam goes on if its score is above -inf (not NaN), a row of logits is read
// if the beam is also not finished.  Both are read at once (the score once more
// where there are no flags).
struct RowState {
    float start;
    bool alive, finished;
};
__device__ inline RowState row_state(const BeamSelect &b, uint32_t row) {
    const int32_t *flags = b.finished ? b.finished : reinterpret_cast<const int32_t *>(b.scores);
    const float start = b.scores[row];
    const int32_t flag = flags[row];
    return {start, start > -INFINITY, b.finished != nullptr && flag != 0};
}

// LDS of best_of, ahead of its short list.
struct BestLds {
    union {
        uint64_t key[kBeamThreads];
        int32_t order[kBeamThreads];
    } most;
    uint32_t count, pad;
};
// Items that the exact selection may list (of four threads for each one wanted,
// or one where more than 64 are), and room for what is read past the last.
constexpr uint32_t kListPad = 32;
constexpr uint32_t best_list(uint32_t best, uint32_t each) { return best * each * (best <= 64 ? 4 : 1) + kListPad; }
constexpr int32_t kNoOrder = INT32_MIN;  // of kNoKey

__device__ inline uint64_t larger_key(uint64_t a, uint64_t b) { return a > b ? a : b; }
template <int CTRL>
__device__ inline int32_t dpp_i32(int32_t x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xF, 0xF, false); }
template <int CTRL>
__device__ inline uint64_t dpp_key(uint64_t k) {
    return static_cast<uint64_t>(static_cast<uint32_t>(dpp_i32<CTRL>(static_cast<int32_t>(k >> 32)))) << 32 |
           static_cast<uint32_t>(dpp_i32<CTRL>(static_cast<int32_t>(k)));
}
template <int CTRL>
__device__ inline double dpp_f64(double x) { return __longlong_as_double(static_cast<long long>(dpp_key<CTRL>(static_cast<uint64_t>(__double_as_longlong(x))))); }
__device__ inline uint64_t lane_key(uint64_t k, int lane) {
    const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(k), lane));
    const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(k >> 32), lane));
    return static_cast<uint64_t>(hi) << 32 | lo;
}
// The least, and the sum, over the 64 lanes, in every lane (see wave_sum).
__device__ inline int32_t wave_least(int32_t v) {
    v = min(v, dpp_i32<0xB1>(v));
    v = min(v, dpp_i32<0x4E>(v));
    v = min(v, dpp_i32<0x124>(v));
    v = min(v, dpp_i32<0x128>(v));
    return min(min(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
               min(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}
__device__ inline float wave_largest(float v) {
    v = fmaxf(v, dpp_f32<0xB1>(v));
    v = fmaxf(v, dpp_f32<0x4E>(v));
    v = fmaxf(v, dpp_f32<0x124>(v));
    v = fmaxf(v, dpp_f32<0x128>(v));
    auto at = [&](int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane)); };
    return fmaxf(fmaxf(at(0), at(16)), fmaxf(at(32), at(48)));
}
__device__ inline double wave_sum(double v) {
    v += dpp_f64<0xB1>(v);
    v += dpp_f64<0x4E>(v);
    v += dpp_f64<0x124>(v);
    v += dpp_f64<0x128>(v);
    auto at = [&](int lane) { return __longlong_as_double(static_cast<long long>(lane_key(static_cast<uint64_t>(__double_as_longlong(v)), lane))); };
    return (at(0) + at(16)) + (at(32) + at(48));
}

// Ranks of the n listed keys: put(rank, key) for the `best` largest.  Up to 64 are
// ranked by four threads each (128 rows by one each: 21.5 us a call against 20.75).
template <class Put>
__device__ inline void rank_list(const uint64_t *list, uint32_t n, uint32_t best, Put put) {
    constexpr uint32_t kShare = 4;
    if (n <= kBeamThreads / kShare) {  // uniform
        const uint32_t c = threadIdx.x / kShare, part = threadIdx.x % kShare;
        if (c >= n) return;
        const uint64_t mine = list[c];
        int32_t rank = 0;
        for (uint32_t j = 0; j < n; j += 8 * kShare) {  // eight reads at a time, the last ones past the end
#pragma unroll
            for (uint32_t u = 0; u < 8; ++u) {
                const uint32_t at = j + u * kShare + part;
                const uint64_t other = list[at];
                rank += at < n && other > mine;
            }
        }
        rank += dpp_i32<0xB1>(rank);
        rank += dpp_i32<0x4E>(rank);
        if (part == 0 && static_cast<uint32_t>(rank) < best) put(static_cast<uint32_t>(rank), mine);
        return;
    }
    for (uint32_t c = threadIdx.x; c < n; c += kBeamThreads) {
        const uint64_t mine = list[c];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < n; j += 8) {
#pragma unroll
            for (uint32_t u = 0; u < 8; ++u) {
                const uint64_t other = list[j + u];
                rank += j + u < n && other > mine;
            }
        }
        if (rank < best) put(rank, mine);
    }
}

// best_of where many items share the order that bounds it (a row masked by one
// low value, say): the same selection by whole keys, of which no two are equal.
template <uint32_t kEach, class Key, class Put>
__device__ inline uint32_t best_exact(uint32_t best, BestLds &lds, uint64_t *list, Key key, Put put) {
    const uint32_t i = threadIdx.x;
    const int lane = i & 63;
    uint64_t own = kNoKey;
#pragma unroll
    for (uint32_t e = 0; e < kEach; ++e) own = larger_key(own, key(e));
    if (i == 0) lds.count = 0;
    uint64_t bound = 1;  // every key
    const uint32_t groups = best <= 64 ? 64 : kBeamThreads;
    if (best <= 64) {
        own = larger_key(own, dpp_key<0xB1>(own));
        own = larger_key(own, dpp_key<0x4E>(own));
        if ((i & 3) == 0) lds.most.key[i >> 2] = own;
    } else {
        lds.most.key[i] = own;
    }
    __syncthreads();
    for (uint32_t q = 0; q < groups; q += 64) {  // every wave ranks them all, one a lane
        const uint64_t mine = lds.most.key[q + lane];
        uint32_t above = 0;
#pragma unroll 8
        for (uint32_t j = 0; j < groups; ++j) above += lds.most.key[j] > mine;
        const uint64_t at = __ballot(mine != kNoKey && above == best - 1);
        if (at != 0) bound = lane_key(mine, __ffsll(static_cast<unsigned long long>(at)) - 1);
    }
#pragma unroll
    for (uint32_t e = 0; e < kEach; ++e) {
        const uint64_t k = key(e);
        if (k >= bound) list[atomicAdd(&lds.count, 1u)] = k;
    }
    __syncthreads();
    const uint32_t n = lds.count;
    rank_list(list, n, best, put);
    return min(n, best);
}

// The `best` largest keys of the workgroup, put(rank, key) for each: key(e) is the
// thread's e-th (kNoKey: none), most its largest order, reaches(bound)(e) whether
// the e-th has at least that order (kNoOrder: none; where orders are near, more may
// be said to, and are listed).  Returns how many there are.  Every thread calls it; LDS is free for the
// next call after a barrier.
//
// The bound is the `best`-th largest of the groups' largest orders, 32 bits; what
// reaches it is listed and ranked by whole keys.  32 groups of 8 threads for up
// to 16 wanted, 64 of 4 for up to 64, else each thread.
template <uint32_t kEach, class Reaches, class Key, class Put>
__device__ inline uint32_t best_of(int32_t most, uint32_t best, BestLds &lds, uint64_t *list, uint32_t room, Reaches reaches, Key key, Put put) {
    const uint32_t i = threadIdx.x;
    const uint32_t lane = i & 63;
    if (i == 0) lds.count = 0;
    const uint32_t groups = best <= 16 ? 32 : (best <= 64 ? 64 : kBeamThreads);
    if (best <= 64) {
        most = max(most, dpp_i32<0xB1>(most));
        most = max(most, dpp_i32<0x4E>(most));
        if (best <= 16) {
            most = max(most, dpp_i32<0x141>(most));  // the other four of eight
            if ((i & 7) == 0) lds.most.order[i >> 3] = most;
        } else if ((i & 3) == 0) {
            lds.most.order[i >> 2] = most;
        }
    } else {
        lds.most.order[i] = most;
    }
    __syncthreads();
    // Every wave ranks the groups: those that fewer than `best` exceed are at least
    // `best`, ties among them, and the least of them is the bound.
    uint32_t members = 0;
    int32_t bound = INT32_MAX;
    for (uint32_t q = 0; q < groups; q += 64) {
        const int32_t mine = q + lane < groups ? lds.most.order[q + lane] : kNoOrder;
        uint32_t above = 0;
        if (groups == 32) {
#pragma unroll
            for (uint32_t j = 0; j < 32; ++j) above += lds.most.order[j] > mine;
        } else {
#pragma unroll 16
            for (uint32_t j = 0; j < groups; ++j) above += lds.most.order[j] > mine;
        }
        const bool in = mine != kNoOrder && above < best;
        members += static_cast<uint32_t>(__popcll(__ballot(in)));
        if (in) bound = min(bound, mine);
    }
    const auto in_list = reaches(members >= best ? wave_least(bound) : kNoOrder + 1);  // or everything
    uint32_t here = 0;
#pragma unroll
    for (uint32_t e = 0; e < kEach; ++e) here += static_cast<uint32_t>(__popcll(__ballot(in_list(e))));
    if (here != 0) {  // uniform over the wave
        uint32_t at = 0;
        if (lane == 0) at = atomicAdd(&lds.count, here);
        at = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(at)));
#pragma unroll
        for (uint32_t e = 0; e < kEach; ++e) {
            const bool mine = in_list(e);
            const uint64_t mask = __ballot(mine);
            if (mask == 0) continue;
            const uint32_t place = at + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
            if (mine && place < room) list[place] = key(e);
            at += static_cast<uint32_t>(__popcll(mask));
        }
    }
    __syncthreads();
    const uint32_t n = lds.count;
    if (n > room) {  // uniform
        __syncthreads();  // everyone has read the count
        return best_exact<kEach>(best, lds, list, key, put);
    }
    rank_list(list, n, best, put);
    return min(n, best);
}
// Keys that best_of lists before it turns to the exact selection.
constexpr uint32_t best_room(uint32_t best) { return best * 4; }

// Grid (segment, row): kBeamSegment logits each.  The logits stay values
// until they are listed: their maximum and what reaches the bound need no more,
// and NaN and masked ones drop out of both.  (Made whole numbers in order first,
// 128 rows 22.9 us a call against 22.1; with 70 registers, seven waves a SIMD, 22.1
// against 21.6.)
__global__ __launch_bounds__(kBeamThreads, 8) void beam_segment_kernel(BeamSelect b) {
    constexpr uint32_t kEach = kBeamEach, kSegment = kBeamSegment;
    extern __shared__ uint64_t list[];
    __shared__ BestLds lds;
    __shared__ float sm_top[kBeamThreads / 64];
    __shared__ double sm_sum[kBeamThreads / 64];
    // Every pointer in one round of scalar loads.
    asm volatile("" ::"s"(b.logits), "s"(b.row_stride), "s"(b.scores), "s"(b.finished), "s"(b.keys), "s"(b.sums), "s"(b.references), "s"(b.arrived));
    const uint32_t segment = blockIdx.x, row = blockIdx.y, i = threadIdx.x;
    // The join's counters, whatever the workspace held: calls of other shapes lay it out differently.
    if (segment == 0 && row < b.batch && i == 0) b.arrived[row] = 0;
    const RowState state = row_state(b, row);
    if (!state.alive || state.finished) return;  // uniform; the row's join reads nothing then
    const float *x = b.logits + static_cast<uint64_t>(row) * b.row_stride;
    const uint32_t first = segment * kSegment;
    float v[kEach];
    if (b.vocab - first >= kSegment) {  // uniform
#pragma unroll
        for (uint32_t c = 0; c < kEach / 4; ++c) {
            const f32x4_any q = __builtin_nontemporal_load(reinterpret_cast<const f32x4_any *>(x + first + (c * kBeamThreads + i) * 4));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[c * 4 + e] = q[e];
        }
    } else {
#pragma unroll
        for (uint32_t e = 0; e < kEach; ++e) {
            const uint32_t at = first + ((e >> 2) * kBeamThreads + i) * 4 + (e & 3);
            v[e] = at < b.vocab ? x[at] : -INFINITY;
        }
    }
    // Largest logit and sum of exponentials of the thread, relative to its own
    // reference, sixteen terms in f32: 15 roundings, 2^-20 of the sum at most, where
    // the terms' own error is 2^-23 and 2^-24 of their distance; all further sums are
    // in 64 bits.  Logits that need cleaning show in one or the other.
    float largest, reference, sum;
    auto scan = [&]() {
        largest = v[0];
#pragma unroll
        for (uint32_t e = 1; e < kEach; ++e) largest = fmaxf(largest, v[e]);
        reference = largest >= -kMostLogit ? largest : 0.f;
        sum = 0.f;
#pragma unroll
        for (uint32_t e = 0; e < kEach; ++e) sum += exp_term(v[e], reference);
    };
    scan();
    if (__any(largest > kMostLogit || sum != sum)) {
#pragma unroll
        for (uint32_t e = 0; e < kEach; ++e) v[e] = clean(v[e]);
        scan();
    }
    // Joined over the wave here, over the waves by the first thread, behind
    // best_of's barrier.
    const bool any = largest >= -kMostLogit;
    const float top = wave_largest(any ? reference : -INFINITY);
    const double total = wave_sum(any ? static_cast<double>(sum * exp_term(reference, top)) : 0.0);
    if ((i & 63) == 0) {
        sm_top[i >> 6] = top;
        sm_sum[i >> 6] = total;
    }
    const size_t part = static_cast<size_t>(row) * b.segments + segment;
    uint64_t *out = b.keys + static_cast<size_t>(row) * b.best * b.segments + segment;
    const uint32_t found = best_of<kEach>(
        any ? order_of(largest) : kNoOrder, b.best, lds, list, best_room(b.best),
        [&](int32_t bound) {  // as values: -0 and +0 are equal then
            const float least = value_of(max(bound, kLeastOrder));
            return [&v, least](uint32_t e) { return v[e] >= least; };
        },
        [&](uint32_t e) {
            return v[e] >= -kMostLogit ? key_of(order_of(v[e]), first + ((e >> 2) * kBeamThreads + i) * 4 + (e & 3)) : kNoKey;
        },
        [&](uint32_t rank, uint64_t key) { out[static_cast<size_t>(rank) * b.segments] = key; });
    for (uint32_t k = found + i; k < b.best; k += kBeamThreads) out[static_cast<size_t>(k) * b.segments] = kNoKey;
    if (i == 0) {
        float all = sm_top[0];
#pragma unroll
        for (uint32_t w = 1; w < kBeamThreads / 64; ++w) all = fmaxf(all, sm_top[w]);
        double s = 0.0;
#pragma unroll
        for (uint32_t w = 0; w < kBeamThreads / 64; ++w)
            if (sm_top[w] > -INFINITY) s += sm_sum[w] * static_cast<double>(exp_term(sm_top[w], all));
        b.references[part] = all;
        b.sums[part] = s;
    }
}

__device__ inline void store_agent(uint64_t *p, uint64_t v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ inline uint64_t load_agent(const uint64_t *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// Keys a thread takes at a time in the join, beside one of the best so far.
constexpr uint32_t kJoinEach = 4;
// The joined lists are sorted and lie rank by rank, the first of each list
// first.  A thread's e-th key: consecutive ones go to different groups of best_of,
// so that the lists' first keys do (lists left whole in a group made the bound so
// low that the exact selection had to follow).
__device__ inline uint32_t join_at(uint32_t e) { return e * kBeamThreads + (threadIdx.x & 7) * (kBeamThreads / 8) + (threadIdx.x >> 3); }

// The `best` largest of keys(0) .. keys(count - 1) into run, in order, kNoKey
// behind.  Every thread calls it, with its first keys, keys(join_at(e)); run is
// complete when it returns, and meanwhile() has run once, while the first waves
// rank a short list.
template <class Keys, class Meanwhile>
__device__ inline void join_keys(uint64_t (&key)[kJoinEach + 1], uint64_t count, uint32_t best, BestLds &lds, uint64_t *list, uint64_t *run, Keys keys,
                                 Meanwhile meanwhile) {
    const uint32_t i = threadIdx.x;
    if (count <= 64 && count <= best_list(best, kJoinEach + 1) - kListPad) {  // uniform: few enough to be ranked as they are (128 are not)
        if (join_at(0) < count) list[join_at(0)] = key[0];
        if (i < best) run[i] = kNoKey;
        __syncthreads();
        rank_list(list, static_cast<uint32_t>(count), best, [&](uint32_t rank, uint64_t k) {
            if (k != kNoKey) run[rank] = k;
        });
        meanwhile();
        __syncthreads();
        return;
    }
    for (uint64_t at = 0; at < count; at += kJoinEach * kBeamThreads) {
        key[kJoinEach] = kNoKey;
        if (at > 0) {
#pragma unroll
            for (uint32_t e = 0; e < kJoinEach; ++e) {
                const uint64_t k = at + join_at(e);
                key[e] = k < count ? keys(k) : kNoKey;
            }
            if (i < best) key[kJoinEach] = run[i];
        }
        int32_t most = kNoOrder;
#pragma unroll
        for (uint32_t e = 0; e <= kJoinEach; ++e) most = max(most, order_in(key[e]));
        const uint32_t found = best_of<kJoinEach + 1>(
            most, best, lds, list, best_room(best), [&](int32_t bound) { return [&key, bound](uint32_t e) { return order_in(key[e]) >= bound; }; },
            [&](uint32_t e) { return key[e]; },
            [&](uint32_t rank, uint64_t k) { run[rank] = k; });
        for (uint32_t k = found + i; k < best; k += kBeamThreads) run[k] = kNoKey;
        if (at == 0) meanwhile();
        __syncthreads();
    }
}

// A workgroup joins the segments of a row; the last row of a batch entry joins
// its rows (relaxed agent-scope stores, their acknowledgement, a counter, and
// agent-scope loads, as the split decode's partitions).
__global__ __launch_bounds__(kBeamThreads) void beam_join_kernel(BeamSelect b) {
    extern __shared__ uint64_t list[];
    __shared__ BestLds lds;
    __shared__ uint64_t run[kBeamMaxBest], run_scores[kBeamMaxBest];
    __shared__ int sm_last;
    __shared__ float sm_most;
    __shared__ double sm_log_sum;
    asm volatile("" ::"s"(b.keys), "s"(b.sums), "s"(b.references), "s"(b.scores), "s"(b.finished), "s"(b.row_keys), "s"(b.row_tokens), "s"(b.arrived));
    asm volatile("" ::"s"(b.next_scores), "s"(b.parents), "s"(b.tokens), "s"(b.next_finished));
    const uint32_t row = blockIdx.x, i = threadIdx.x, entry = row / b.beams;
    const size_t part = static_cast<size_t>(row) * b.segments;
    const uint64_t *keys = b.keys + part * b.best;  // [rank][segment]
    const uint64_t count = static_cast<uint64_t>(b.segments) * b.best;
    // All first loads together (of a row that was not read, whatever is there).
    uint64_t key_in[kJoinEach + 1];
#pragma unroll
    for (uint32_t e = 0; e < kJoinEach; ++e) key_in[e] = keys[min(static_cast<uint64_t>(join_at(e)), count - 1)];
    const uint32_t lane = i & 63, s0 = min(lane, b.segments - 1);
    const float reference0 = b.references[part + s0];
    const double sum0 = b.sums[part + s0];
    const RowState state = row_state(b, row);
    const float start = state.start;
    const bool finished = state.finished, alive = state.alive;
    if (alive && !finished) {  // uniform
#pragma unroll
        for (uint32_t e = 0; e < kJoinEach; ++e)
            if (join_at(e) >= count) key_in[e] = kNoKey;
        join_keys(key_in, count, b.best, lds, list, run, [&](uint64_t k) { return keys[k]; }, [&]() {
            if (i < kBeamThreads - 64) return;
            // The last wave sums the segments (0.65 us, of which the ranks cover a half).
            float most = -INFINITY;
            for (uint32_t s = lane; s < b.segments; s += 64) most = fmaxf(most, s == lane ? reference0 : b.references[part + s]);
            most = wave_largest(most);
            double log_sum = 0.0;
            if (most > -INFINITY) {  // uniform: something is not masked
                double sum = 0.0;
                for (uint32_t s = lane; s < b.segments; s += 64)
                    sum += (s == lane ? sum0 : b.sums[part + s]) * exp(static_cast<double>(s == lane ? reference0 : b.references[part + s]) - most);
                log_sum = log(wave_sum(sum));
            }
            if (lane == 0) {
                sm_most = most;
                sm_log_sum = log_sum;
            }
        });
    } else {
        for (uint32_t k = i; k < b.best; k += kBeamThreads)
            run[k] = alive && k == 0 ? key_of(0, static_cast<uint32_t>(b.end_token)) : kNoKey;
        __syncthreads();
    }
    // Thread i holds rank i of the row: its token, and its score's key.
    const uint32_t beam = row - entry * b.beams;
    uint64_t key = kNoKey, scored = kNoKey;
    double score = 0.0;
    if (i < b.best) {
        key = run[i];
        score = finished ? static_cast<double>(start) : start + ((static_cast<double>(value_of(order_in(key))) - static_cast<double>(sm_most)) - sm_log_sum);
        if (key != kNoKey) scored = score_key(score, beam * b.best + i);
    }
    const size_t rows_at = static_cast<size_t>(entry) * b.beams * b.best, at = rows_at + static_cast<size_t>(i) * b.beams + beam;  // [rank][beam]
    if (b.beams > 1) {
        if (i < b.best) {
            store_agent(b.row_keys + at, scored);
            store_agent(b.row_tokens + at,
                        static_cast<uint64_t>(token_in(key)) << 32 | __float_as_uint(static_cast<float>(score)));
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (i == 0) sm_last = __hip_atomic_fetch_add(b.arrived + entry, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == b.beams - 1;
        __syncthreads();
        if (!sm_last) return;
        const uint64_t all = static_cast<uint64_t>(b.beams) * b.best;
        auto scores = [&](uint64_t k) { return load_agent(b.row_keys + rows_at + k); };
#pragma unroll
        for (uint32_t e = 0; e < kJoinEach; ++e) key_in[e] = join_at(e) < all ? scores(join_at(e)) : kNoKey;
        join_keys(key_in, all, b.best, lds, list, run_scores, scores, []() {});
        if (i >= b.best) return;
        scored = run_scores[i];
    }
    if (i >= b.best) return;
    const size_t o = static_cast<size_t>(entry) * b.best + i;
    int32_t parent = -1, token = -1, ended = 0;
    float value = -INFINITY;
    if (scored != kNoKey) {
        const uint32_t number = number_in(scored), from = number / b.best;
        parent = static_cast<int32_t>(entry * b.beams + from);
        if (b.beams > 1) {
            const uint64_t held = load_agent(b.row_tokens + rows_at + static_cast<size_t>(number - from * b.best) * b.beams + from);
            token = static_cast<int32_t>(held >> 32);
            value = __uint_as_float(static_cast<uint32_t>(held));
        } else {
            token = static_cast<int32_t>(token_in(key));
            value = static_cast<float>(score);
        }
        ended = token == b.end_token || (b.finished != nullptr && b.finished[parent] != 0);
    }
    b.next_scores[o] = value;
    b.parents[o] = parent;
    b.tokens[o] = token;
    if (b.next_finished) b.next_finished[o] = ended;
}

}  // namespace

int launch_beam_select(const BeamSelect &b, void *stream) {
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid(b.segments, b.batch * b.beams);
    hipLaunchKernelGGL(beam_segment_kernel, grid, dim3(kBeamThreads), best_list(b.best, kBeamEach) * 8, st, b);
    hipLaunchKernelGGL(beam_join_kernel, dim3(b.batch * b.beams), dim3(kBeamThreads), best_list(b.best, kJoinEach + 1) * 8, st, b);
    return static_cast<int>(hipGetLastError());
}

}  // namespace pvlc
