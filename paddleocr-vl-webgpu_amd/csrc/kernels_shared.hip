// One decode step of groups of sequences that share their first pages: the shared
// rows are attended once for all of a group, each sequence's own rows by
// themselves, and the parts joined.  The new rows are in the pages by then.

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "attend_device.hpp"

namespace pvlc {
namespace {

constexpr int kWaves = kSharedWaves, kThreads = kWaves * 64;

// A group's set of up to 2 CT sequences, a share of find_share: 16 columns are
// the 8 heads of a kv head of 2 sequences.
template <int CT>
struct SharedSet {
    int first, count;  // sequences
    int shared;        // rows, in whole blocks
};

// The rows that a group shares are no more than its shortest sequence has.
// Sequences whose length does not fit the call are left out (the append reports
// them, and so it does offsets that are none).
template <int CT>
__device__ inline bool find_set(const SharedRows &p, uint32_t u, SharedSet<CT> *set) {
    RaggedRows groups = p.ragged;
    groups.num_seqs = p.num_groups;
    groups.rows = p.ragged.num_seqs;
    groups.each = p.ragged.num_seqs / p.num_groups;
    groups.offsets = p.group_offsets;
    groups.lens = p.shared_lens;
    groups.max_tokens = 0xFFFFFFFFu;
    const SeqRows q = find_share<2 * CT, 1>(groups, u);
    const int first = q.share * 2 * CT;
    if (!q.ok || first >= q.count) {
        if (!q.ok && threadIdx.x == 0) atomicOr(p.error_word, 1u);
        return false;
    }
    const int lane = threadIdx.x & 63;
    int least = q.held;
    for (int i = lane; i < q.count; i += 64) {
        const int len = p.ragged.lens[q.begin + i];
        if (len >= 0 && static_cast<uint32_t>(len) < p.ragged.max_tokens) least = min(least, len);
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) least = min(least, __shfl_xor(least, d));
    set->first = q.begin + first;
    set->count = min(q.count - first, 2 * CT);
    set->shared = __builtin_amdgcn_readfirstlane(least) / static_cast<int>(kBlockTokens) * static_cast<int>(kBlockTokens);
    return true;
}

__device__ inline bool fits(const SharedRows &p, int len) { return len >= 0 && static_cast<uint32_t>(len) < p.ragged.max_tokens; }

// Steps of a part: the keys are cut into `parts` (fewer for few keys: a part has a step for each wave).
__device__ inline int part_steps(int keys, int parts) {
    const int steps = (keys + kAttendStep - 1) / kAttendStep;
    return max((steps + parts - 1) / parts, kWaves);
}

// CT * 16 columns over the part's steps, a wave every fourth step; the waves' results joined through LDS, and written unnormalised.
template <int CODE, bool F32, int CT>
__device__ inline void attend_part(const SharedRows &p, int seq0, int rows, int columns, uint32_t g, AttendPages pages, int keys, int first,
                                   int end, float *part_o, float *part_ml, float (*sm_m)[64], float (*sm_l)[64], float4_t *sm_o) {
    typedef std::conditional_t<F32, float, uint16_t> Element;
    const int lane = threadIdx.x & 63, row = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    half8_t qf[CT][4];
    int limit[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        const int seq = seq0 + min(ct * 2 + (row >> 3), rows - 1);
        const int64_t pos = p.positions ? p.positions[seq] : p.ragged.lens[seq];
        const bool rope = p.rotate_query && p.rope_cos != nullptr && pos >= 0 && pos < static_cast<int64_t>(p.rope_rows);
        const Element *src = static_cast<const Element *>(p.query) + (static_cast<int64_t>(seq) * kQueryHeads + g * kGroup + (row & 7)) * kHeadDim;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            AttendQuery<F32> raw;
            raw.load(src, attend_dim<CODE>(kb, kg));
            float4_t cs[2]{}, sn[2]{};
            if (rope) {
#pragma unroll
                for (int f = 0; f < 2; ++f) {
                    cs[f] = *reinterpret_cast<const float4_t *>(p.rope_cos + pos * 64 + attend_dim<CODE>(kb, kg) + f * 4);
                    sn[f] = *reinterpret_cast<const float4_t *>(p.rope_sin + pos * 64 + attend_dim<CODE>(kb, kg) + f * 4);
                }
            }
            raw.rotate(rope, cs, sn, &qf[ct][kb], &qf[ct][kb + 2]);
        }
        limit[ct] = keys;
    }
    pages.keys = static_cast<const uint8_t *>(p.key_cache);
    pages.values = static_cast<const uint8_t *>(p.value_cache);
    pages.exponents = p.exponents;
    pages.num_blocks = p.ragged.num_blocks;
    pages.head = g;
    pages.last_tile = (keys - 1) >> 4;
    AttendState<CT> st;
    st.clear();
    attend<CODE, F32, CT>(pages, qf, first + wave, end, kWaves, keys / kAttendStep, limit, keys, p.scale_log2, st);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        const float l = column_sum(st.l[ct]);
        if (kg == 0) {
            sm_m[wave][ct * 16 + row] = st.m[ct];
            sm_l[wave][ct * 16 + row] = l;
        }
    }
    __syncthreads();
    float a[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        float m = sm_m[0][ct * 16 + row];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) m = fmaxf(m, sm_m[w][ct * 16 + row]);
        a[ct] = st.m[ct] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((st.m[ct] - m) * p.scale_log2);
    }
    for (int c = static_cast<int>(threadIdx.x); c < columns; c += kThreads) {
        float m = sm_m[0][c], l = 0.f;
#pragma unroll
        for (int w = 1; w < kWaves; ++w) m = fmaxf(m, sm_m[w][c]);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) l += sm_m[w][c] == -INFINITY ? 0.f : sm_l[w][c] * __builtin_amdgcn_exp2f((sm_m[w][c] - m) * p.scale_log2);
        part_ml[c * 2] = m * p.scale_log2;
        part_ml[c * 2 + 1] = l;
    }
    // Two 16-dim tiles at a time.
#pragma unroll
    for (int c0 = 0; c0 < 8; c0 += 2) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) sm_o[((wave * 2 + c) * CT + ct) * 64 + lane] = st.o[ct][c0 + c] * a[ct];
        __syncthreads();
        for (int i = static_cast<int>(threadIdx.x); i < 2 * CT * 64; i += kThreads) {
            const int l = i & 63, ct = (i >> 6) % CT, c = (i >> 6) / CT, column = ct * 16 + (l & 15);
            float4_t v = sm_o[i];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) v += sm_o[w * 2 * CT * 64 + i];
            if (column < columns) *reinterpret_cast<float4_t *>(part_o + column * kHeadDim + (c0 + c) * 16 + (l >> 4) * 4) = v;
        }
        __syncthreads();
    }
}

// Workgroup: share u, kv head, then the parts of the shared rows and those of
// the set's sequences.
template <int CODE, bool F32, int CT>
__global__ __launch_bounds__(kThreads, CT == 4 ? 1 : 2) void shared_attention_kernel(SharedRows p) {
    __shared__ float sm_m[kWaves][64], sm_l[kWaves][64];
    __shared__ float4_t sm_o[kWaves * 2 * CT * 64];
    const uint32_t g = blockIdx.x & 1u;
    uint32_t b = blockIdx.x >> 1;
    const bool common = b < p.shares * p.shared_parts;  // uniform
    if (!common) b -= p.shares * p.shared_parts;
    const uint32_t per = common ? p.shared_parts : 2 * CT * p.own_parts;
    const uint32_t u = b / per, rest = b % per;
    SharedSet<CT> set;
    if (!find_set<CT>(p, u, &set)) return;
    AttendPages pages{};
    if (common) {
        const int steps = part_steps(set.shared, static_cast<int>(p.shared_parts)), first = static_cast<int>(rest) * steps;
        if (first * kAttendStep >= set.shared) return;
        pages.table = p.ragged.tables + static_cast<size_t>(set.first) * p.ragged.max_blocks;
        const size_t slot = (static_cast<size_t>(u) * 2 + g) * p.shared_parts + rest;
        attend_part<CODE, F32, CT>(p, set.first, set.count, set.count * static_cast<int>(kGroup), g, pages, set.shared, first,
                                   min(first + steps, (set.shared + kAttendStep - 1) / kAttendStep),
                                   p.part_o + slot * CT * 16 * kHeadDim, p.part_ml + slot * CT * 16 * 2, sm_m, sm_l, sm_o);
    } else {
        const int r = static_cast<int>(rest / p.own_parts), part = static_cast<int>(rest % p.own_parts);
        if (r >= set.count) return;
        const int seq = set.first + r, len = p.ragged.lens[seq];
        if (!fits(p, len)) return;
        const int keys = len + 1 - set.shared, steps = part_steps(keys, static_cast<int>(p.own_parts)), first = part * steps;
        if (first * kAttendStep >= keys) return;
        pages.table = p.ragged.tables + static_cast<size_t>(seq) * p.ragged.max_blocks + set.shared / static_cast<int>(kBlockTokens);
        const size_t slot = ((static_cast<size_t>(u) * 2 + g) * 2 * CT + r) * p.own_parts + part;
        attend_part<CODE, F32, 1>(p, seq, 1, kGroup, g, pages, keys, first, min(first + steps, (keys + kAttendStep - 1) / kAttendStep),
                                  p.own_o + slot * kGroup * kHeadDim, p.own_ml + slot * kGroup * 2, sm_m, sm_l, sm_o);
    }
}

// Workgroup: a sequence and kv head; thread t has head t / 32 and dims t % 32 * 4 .. + 3.
template <bool F32, int CT>
__global__ __launch_bounds__(256) void shared_merge_kernel(SharedRows p) {
    const uint32_t g = blockIdx.x & 1u, u = (blockIdx.x >> 1) / (2 * CT);
    const int r = static_cast<int>((blockIdx.x >> 1) % (2 * CT));
    SharedSet<CT> set;
    if (!find_set<CT>(p, u, &set) || r >= set.count) return;
    const int seq = set.first + r, len = p.ragged.lens[seq];
    if (!fits(p, len)) return;
    const int head = threadIdx.x >> 5, d0 = (threadIdx.x & 31) * 4;
    auto parts_of = [](int keys, uint32_t parts) {
        const int steps = part_steps(keys, static_cast<int>(parts));
        return keys <= 0 ? 0 : ((keys + kAttendStep - 1) / kAttendStep + steps - 1) / steps;
    };
    const int shared = parts_of(set.shared, p.shared_parts), own = parts_of(len + 1 - set.shared, p.own_parts);
    const size_t unit = static_cast<size_t>(u) * 2 + g;
    float m = -INFINITY, l = 0.f;
    float4_t o{0.f, 0.f, 0.f, 0.f};
    auto add = [&](const float *ml, const float *po) {
        const float pm = ml[0], pl = ml[1];
        const float4_t v = *reinterpret_cast<const float4_t *>(po);
        const float top = fmaxf(m, pm);
        const float a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top), b = pm == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(pm - top);
        l = l * a + pl * b;
        o = o * a + v * b;
        m = top;
    };
    for (int i = 0; i < shared; ++i) {
        const size_t column = (unit * p.shared_parts + i) * CT * 16 + r * kGroup + head;
        add(p.part_ml + column * 2, p.part_o + column * kHeadDim + d0);
    }
    for (int i = 0; i < own; ++i) {
        const size_t column = ((unit * 2 * CT + r) * p.own_parts + i) * kGroup + head;
        add(p.own_ml + column * 2, p.own_o + column * kHeadDim + d0);
    }
    const float inv = 1.0f / l;
    const size_t at = (static_cast<size_t>(seq) * kQueryHeads + g * kGroup + head) * kHeadDim + d0;
    if constexpr (F32) *reinterpret_cast<float4_t *>(static_cast<float *>(p.out) + at) = o * inv;
    else *reinterpret_cast<half4_t *>(static_cast<uint16_t *>(p.out) + at) = half4_t{to_h(o[0] * inv), to_h(o[1] * inv), to_h(o[2] * inv), to_h(o[3] * inv)};
}

template <int CODE, bool F32, int CT>
void launch(const SharedRows &p, hipStream_t stream) {
    const uint32_t groups = 2 * p.shares * (p.shared_parts + 2 * CT * p.own_parts);
    hipLaunchKernelGGL((shared_attention_kernel<CODE, F32, CT>), dim3(groups), dim3(kThreads), 0, stream, p);
    hipLaunchKernelGGL((shared_merge_kernel<F32, CT>), dim3(2 * p.shares * 2 * CT), dim3(256), 0, stream, p);
}

template <int CODE, bool F32>
void launch_columns(const SharedRows &p, hipStream_t stream) {
    if (p.columns == 1) launch<CODE, F32, 1>(p, stream);
    else if (p.columns == 2) launch<CODE, F32, 2>(p, stream);
    else launch<CODE, F32, 4>(p, stream);
}

template <bool F32>
void launch_code(const SharedRows &p, hipStream_t stream) {
    if (p.code == PVLC_HIP_KV_F16) launch_columns<PVLC_HIP_KV_F16, F32>(p, stream);
    else if (p.code == PVLC_HIP_KV_E4M3) launch_columns<PVLC_HIP_KV_E4M3, F32>(p, stream);
    else launch_columns<PVLC_HIP_KV_INT8, F32>(p, stream);
}

}  // namespace

int launch_shared_decode(const SharedRows &rows, void *stream) {
    SharedRows p = rows;
    p.scale_log2 = kAttendLog2e / sqrtf(static_cast<float>(kHeadDim));
    if (p.f32) launch_code<true>(p, static_cast<hipStream_t>(stream));
    else launch_code<false>(p, static_cast<hipStream_t>(stream));
    return static_cast<int>(hipGetLastError());
}

}  // namespace pvlc
