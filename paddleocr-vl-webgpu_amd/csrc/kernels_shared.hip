// One decode step of groups of sequences that share their first pages: the shared
// rows are attended once for all of a group, each sequence's own rows by
// themselves, and the parts joined by a second launch.
//
// With m, l, o the largest score, the sum of weights exp(score - m) and their sum of
// values over any part of a sequence's rows, parts join as
//   m = max m_p,  out = sum_p exp(m_p - m) o_p / sum_p exp(m_p - m) l_p.
//
// A part whose scores are all NaN has the reference of one without keys, -infinity, and a
// sum of NaN: parts join by products with a factor of 0, which keep it, and are never left out.
//
// Bytes are what a group's shared rows take once, so large calls are bound by
// memory: 32 groups of eight sequences on 8192 to 32768 shared rows (fp16, 607 MB) 150
// us, 4.0 TB/s of a copy's 5.1.  A group of more than four sequences is several sets,
// each of which reads the rows again, from the XCD's L2 (the parts are a multiple of four,
// which puts a part of every set of a group on one XCD), and converts 8-bit codes
// again: 64 sequences on 16384 rows (int8, f32 operands) 41 us where the products
// take 16.  Small calls are bound by two launches of dependent rounds: 16 groups of
// eight on 300 to 2010 rows (e4m3) 17.2 us.  Measured and not kept: sets of eight
// sequences (512 registers, one workgroup a compute unit: those 16 groups 55 us against
// 29 then), the join by the workgroup that comes last (33 against 29, one group of four
// 15.9 against 13.2), parts for 384 / 512 / 1024 workgroups in place of 256 (the 64
// sequences 46 / 44 / 50, the 16 groups 22 / 22 / 22).

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "attend_device.hpp"

namespace pvlc {
namespace {

constexpr int kWaves = kSharedWaves, kThreads = kWaves * 64;

// Up to 2 CT sequences of a group: 16 columns are the 8 heads of a kv head of 2 sequences.
struct SharedSet {
    int first, count;  // sequences
    int shared;        // rows, in whole blocks (0 where no sequence of the set fits)
    int through;       // of the set's sequences, the first that fits: its table has the shared blocks
    int lens;          // lane i: the length of sequence i
    __device__ int len(int i) const { return __builtin_amdgcn_readlane(lens, i); }
};

__device__ inline bool fits(const SharedRows &p, int len) { return len >= 0 && static_cast<uint32_t>(len) < p.ragged.max_tokens; }

// The rows that a group shares are no more than its shortest sequence has.
// Sequences whose length does not fit the call are left out (they are reported
// where their row would be appended); a set of none else shares nothing, whatever
// the shared length says: nothing would keep that within the table.
template <int CT>
__device__ inline bool find_set(const SharedRows &p, uint32_t u, SharedSet *set) {
    int begin, count, first, least;
    if (p.group_offsets) {
        RaggedRows groups = p.ragged;
        groups.num_seqs = p.num_groups;
        groups.rows = p.ragged.num_seqs;
        groups.offsets = p.group_offsets;
        groups.lens = p.shared_lens;
        groups.max_tokens = 0xFFFFFFFFu;
        const SeqRows q = find_share<2 * CT, 1>(groups, u);
        first = q.share * 2 * CT;
        if ((!q.ok || q.told) && threadIdx.x == 0) atomicOr(p.error_word, 1u);
        if (!q.ok || first >= q.count) return false;
        begin = q.begin;
        count = q.count;
        least = q.held;
    } else {
        count = static_cast<int>(p.ragged.num_seqs / p.num_groups);
        const int sets = (count + 2 * CT - 1) / (2 * CT), group = static_cast<int>(u) / sets;
        first = (static_cast<int>(u) - group * sets) * 2 * CT;
        begin = group * count;
        least = p.shared_lens[group];
    }
    const int lane = threadIdx.x & 63;
    set->first = begin + first;
    set->count = min(count - first, 2 * CT);
    set->lens = p.ragged.lens[set->first + min(lane, set->count - 1)];
    for (int i = lane; i < count; i += 64) {
        const int len = p.ragged.lens[begin + i];
        if (fits(p, len)) least = min(least, len);
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) least = min(least, __shfl_xor(least, d));
    least = __builtin_amdgcn_readfirstlane(least);
    if (least < 0) {
        if (threadIdx.x == 0) atomicOr(p.error_word, 1u);
        return false;
    }
    const uint64_t mine = __ballot(lane < set->count && fits(p, set->lens));
    set->through = mine ? __builtin_ctzll(mine) : 0;
    set->shared = mine ? least / static_cast<int>(kBlockTokens) * static_cast<int>(kBlockTokens) : 0;
    return true;
}

// Steps of a part: the keys are cut into `parts`, fewer for few keys (a part has
// `least` steps: one for each wave of shared rows, two of own ones); and the
// parts that this makes.
constexpr int kLeastShared = kWaves, kLeastOwn = 2;
__device__ inline int part_steps(int keys, int parts, int least) { return max(((keys + kAttendStep - 1) / kAttendStep + parts - 1) / parts, least); }
__device__ inline int parts_of(int keys, int parts, int least) {
    const int steps = part_steps(keys, parts, least);
    return ((keys + kAttendStep - 1) / kAttendStep + steps - 1) / steps;
}

// A wave's results: of its columns, reference, sum and outputs [16-dim tile][16 columns][lane].
template <int CT>
struct SharedLds {
    float m[kWaves][CT * 16], l[kWaves][CT * 16];
    float4_t o[kWaves][8 * CT * 64];
};

// cos and sin of the 8 dims from d0 (below 64) at a position.
__device__ inline void load_angles(const SharedRows &p, bool rope, int64_t pos, int d0, float4_t (&cs)[2], float4_t (&sn)[2]) {
#pragma unroll
    for (int f = 0; f < 2; ++f) {
        cs[f] = rope ? *reinterpret_cast<const float4_t *>(p.rope_cos + pos * 64 + d0 + f * 4) : float4_t{};
        sn[f] = rope ? *reinterpret_cast<const float4_t *>(p.rope_sin + pos * 64 + d0 + f * 4) : float4_t{};
    }
}

// The new row of a sequence, by one wave: rotated, written to its page, and one
// more key of the wave's columns.
template <bool F32>
__device__ inline void append_and_attend(const SharedRows &p, int seq, int len, uint32_t g, const half8_t (&qf)[4], AttendState<1> &st) {
    typedef std::conditional_t<F32, float, uint16_t> Element;
    constexpr int kF16 = PVLC_HIP_KV_F16;
    const int lane = threadIdx.x & 63, row = lane & 15, kg = lane >> 4;
    const size_t at = (static_cast<size_t>(seq) * kKvHeads + g) * kHeadDim;
    const Element *key = static_cast<const Element *>(p.new_key) + at, *value = static_cast<const Element *>(p.new_value) + at;
    const int64_t pos = p.positions ? p.positions[seq] : len;
    const bool rope = p.rope_cos != nullptr && pos >= 0 && pos < static_cast<int64_t>(p.rope_rows);
    const int64_t id = p.ragged.tables[static_cast<size_t>(seq) * p.ragged.max_blocks + len / static_cast<int>(kBlockTokens)];
    half8_t k[4];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
        AttendQuery<F32> raw;
        float4_t cs[2], sn[2];
        raw.load(key, attend_dim<kF16>(kb, kg));
        load_angles(p, rope, pos, attend_dim<kF16>(kb, kg), cs, sn);
        raw.rotate(rope, cs, sn, &k[kb], &k[kb + 2]);
        if constexpr (!F32) {
            if (!rope) {  // as given, bit for bit
                k[kb] = raw.x[0][0];
                k[kb + 2] = raw.x[1][0];
            }
        }
    }
    auto half_value = [&](int d) { return F32 ? to_h(value[d]) : __builtin_bit_cast(_Float16, static_cast<uint16_t>(value[d])); };
    bool ok;
    const size_t slab = (static_cast<size_t>(checked_block(p.ragged, id, &ok)) * kKvHeads + g) * kBlockHeadElems;
    const int slot = len % static_cast<int>(kBlockTokens);
    if (ok) {
        uint16_t *kc = static_cast<uint16_t *>(p.key_cache) + slab + key_slot(slot) * 8;
        if (row == 0) {
#pragma unroll
            for (int kb = 0; kb < 4; ++kb) *reinterpret_cast<half8_t *>(kc + attend_dim<kF16>(kb, kg) / 8 * 128) = k[kb];
        }
        uint16_t *vc = static_cast<uint16_t *>(p.value_cache) + slab + slot;
#pragma unroll
        for (int d = 0; d < 2; ++d) vc[(lane + d * 64) * kBlockTokens] = __builtin_bit_cast(uint16_t, half_value(lane + d * 64));
    }
    if (lane == 0 && g == 0) {
        if (!ok) atomicOr(p.error_word, 2u);
        if (!rope && p.rope_cos != nullptr) atomicOr(p.error_word, 4u);
    }
    // Key 0 of a score product whose other rows are 0.
    float4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(row == 0 ? k[kb] : half8_t{}, qf[kb], acc, 0, 0, 0);
    const float x = __shfl(acc[0], row), top = fmaxf(st.m[0], x);
    const float a = st.m[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((st.m[0] - top) * p.scale_log2);
    const float w = x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((x - top) * p.scale_log2);  // (it may be the only key so far)
    st.m[0] = top;
    st.l[0] = st.l[0] * a + (kg == 0 ? w : 0.f);
#pragma unroll
    for (int c = 0; c < 8; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) st.o[0][c][r] = st.o[0][c][r] * a + w * static_cast<float>(half_value(c * 16 + kg * 4 + r));
}

// The new row of a sequence into its 8-bit block, by the one wave that reads this
// block: two dims a lane, as the paged decode appends its own.  Complete, and seen by
// the wave's loads, when this returns.
template <int CODE, bool F32>
__device__ inline void append_q8(const SharedRows &p, int seq, int len, uint32_t g) {
    typedef std::conditional_t<F32, float, uint16_t> Element;
    const int lane = threadIdx.x & 63, slot = len % static_cast<int>(kBlockTokens);
    const size_t at = (static_cast<size_t>(seq) * kKvHeads + g) * kHeadDim + lane;
    const Element *key = static_cast<const Element *>(p.new_key) + at, *value = static_cast<const Element *>(p.new_value) + at;
    auto given = [](Element x) { return F32 ? static_cast<float>(x) : static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(x))); };
    const Element kl = key[0], kh = key[64], vl = value[0], vh = value[64];
    const int64_t pos = p.positions ? p.positions[seq] : len;
    const bool rope = p.rope_cos != nullptr && pos >= 0 && pos < static_cast<int64_t>(p.rope_rows);
    const float c = rope ? p.rope_cos[pos * 64 + lane] : 1.f, s = rope ? p.rope_sin[pos * 64 + lane] : 0.f;
    bool ok;
    const size_t slab = static_cast<size_t>(checked_block(p.ragged, p.ragged.tables[static_cast<size_t>(seq) * p.ragged.max_blocks + len / static_cast<int>(kBlockTokens)], &ok)) * kKvHeads + g;
    const uint32_t old = *reinterpret_cast<const uint16_t *>(p.exponents + slab * 2);
    if (lane == 0 && g == 0) {
        if (!ok) atomicOr(p.error_word, 2u);
        if (!rope && p.rope_cos != nullptr) atomicOr(p.error_word, 4u);
    }
    if (!ok) return;  // uniform
    float k_lo = given(kl), k_hi = given(kh);
    if (rope) {
        const float x = k_lo;
        k_lo = x * c + (-k_hi) * s;
        k_hi = k_hi * c + x * s;
    }
    auto held = [](float x) { return q8_value(static_cast<float>(to_h(x))); };
    k_lo = held(k_lo);
    k_hi = held(k_hi);
    const float v_lo = held(given(vl)), v_hi = held(given(vh));
    const int old_k = static_cast<int>(old & 255) - kQ8Bias, old_v = static_cast<int>(old >> 8) - kQ8Bias;
    int e_k = q8_exponent<CODE>(wave_max(q8_size(q8_size(0.f, k_lo), k_hi)));
    int e_v = q8_exponent<CODE>(wave_max(q8_size(q8_size(0.f, v_lo), v_hi)));
    if (slot > 0) {
        e_k = max(e_k, old_k);
        e_v = max(e_v, old_v);
    }
    const float pk = exp2_whole(-e_k), pv = exp2_whole(-e_v);
    const uint32_t codes = q8_encode<CODE>(k_lo * pk, k_hi * pk, v_lo * pv, v_hi * pv);
    uint8_t *ks = static_cast<uint8_t *>(p.key_cache) + slab * kQ8SlabBytes, *vs = static_cast<uint8_t *>(p.value_cache) + slab * kQ8SlabBytes;
    const int grown = __builtin_amdgcn_readfirstlane(slot > 0 ? (e_k - old_k) | (e_v - old_v) << 16 : 0);
    if (grown != 0) requantise_block<CODE>(ks, vs, lane, slot, grown & 0xFFFF, grown >> 16);
    // key (slot, d) at (slot/4)*512 + (d/16)*64 + (slot%4)*16 + d%16, value at d*16 + slot
    uint8_t *kd = ks + (slot >> 2) * 512 + (slot & 3) * 16 + (lane >> 4) * 64 + (lane & 15), *vd = vs + lane * 16 + slot;
    kd[0] = static_cast<uint8_t>(codes);
    kd[256] = static_cast<uint8_t>(codes >> 8);
    vd[0] = static_cast<uint8_t>(codes >> 16);
    vd[1024] = static_cast<uint8_t>(codes >> 24);
    if (lane == 0) *reinterpret_cast<uint16_t *>(p.exponents + slab * 2) = static_cast<uint16_t>((e_k + kQ8Bias) | (e_v + kQ8Bias) << 8);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
}

// Eight dims of a lane's column (the query of head row & 7 of sequence r of the
// set) and their rotary partners: sent for, then rotated.
template <int CODE, bool F32>
struct SharedQuery {
    AttendQuery<F32> raw;
    float4_t cs[2], sn[2];
    bool rope;
    __device__ __attribute__((always_inline)) void send(const SharedRows &p, const SharedSet &set, int r, uint32_t g, int kb) {
        const int lane = threadIdx.x & 63, row = lane & 15, kg = lane >> 4, seq = set.first + r, len = __shfl(set.lens, r);
        const int64_t pos = p.positions ? p.positions[seq] : len;
        rope = p.rotate_query && p.rope_cos != nullptr && pos >= 0 && pos < static_cast<int64_t>(p.rope_rows);
        const auto *src = static_cast<const typename AttendQuery<F32>::Element *>(p.query) +
                          (static_cast<int64_t>(seq) * kQueryHeads + g * kGroup + (row & 7)) * kHeadDim;
        raw.load(src, attend_dim<CODE>(kb, kg));
        load_angles(p, rope, pos, attend_dim<CODE>(kb, kg), cs, sn);
    }
    __device__ __attribute__((always_inline)) void take(half8_t *lo, half8_t *hi) const { raw.rotate(rope, cs, sn, lo, hi); }
};

__device__ inline AttendPages pages_of(const SharedRows &p, int seq, int first_row, int keys, uint32_t g) {
    AttendPages pages;
    pages.keys = static_cast<const uint8_t *>(p.key_cache);
    pages.values = static_cast<const uint8_t *>(p.value_cache);
    pages.exponents = p.exponents;
    pages.table = p.ragged.tables + static_cast<size_t>(seq) * p.ragged.max_blocks + first_row / static_cast<int>(kBlockTokens);
    pages.first = 0;
    pages.num_blocks = p.ragged.num_blocks;
    pages.head = g;
    pages.last_tile = (keys - 1) >> 4;
    return pages;
}

// A part of a set's shared rows: the columns of all its sequences, a wave every
// fourth step; the waves' results joined through LDS, and written unnormalised.
template <int CODE, bool F32, int CT>
__device__ inline void attend_shared(const SharedRows &p, const SharedSet &set, uint32_t g, int first, int end, float *part_o, float *part_ml,
                                     SharedLds<CT> &lds) {
    const int lane = threadIdx.x & 63, row = lane & 15, kg = lane >> 4, columns = set.count * static_cast<int>(kGroup), keys = set.shared;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    // Wave w rotates pair w % 2 of column tile w / 2; all take the rest from LDS.
    SharedQuery<CODE, F32> query;
    if (wave < 2 * CT) query.send(p, set, min((wave >> 1) * 2 + (row >> 3), set.count - 1), g, wave & 1);
    __builtin_amdgcn_sched_barrier(0);
    Attend<CODE, F32, CT> loop;
    loop.begin(pages_of(p, set.first + set.through, 0, keys, g), first + wave, end, kWaves);
    half8_t *const sm_q = reinterpret_cast<half8_t *>(&lds.o[0][0]);  // [column tile][kb][lane], before the join
    if (wave < 2 * CT) {
        half8_t lo, hi;
        query.take(&lo, &hi);
        sm_q[((wave >> 1) * 4 + (wave & 1)) * 64 + lane] = lo;
        sm_q[((wave >> 1) * 4 + (wave & 1) + 2) * 64 + lane] = hi;
    }
    // (fences of LDS alone: the keys and values stay in flight)
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    half8_t qf[CT][4];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) qf[ct][kb] = sm_q[(ct * 4 + kb) * 64 + lane];
    int limit[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) limit[ct] = keys;
    AttendState<CT> st;
    st.clear();
    loop.run(qf, keys / kAttendStep, limit, keys, p.scale_log2, st);
    if (loop.bad && lane == 0) atomicOr(p.error_word, 2u);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        const float l = column_sum(st.l[ct]);
        if (kg == 0) {
            lds.m[wave][ct * 16 + row] = st.m[ct];
            lds.l[wave][ct * 16 + row] = l;
        }
    }
    __syncthreads();
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        float m = lds.m[0][ct * 16 + row];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) m = fmaxf(m, lds.m[w][ct * 16 + row]);
        const float a = st.m[ct] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((st.m[ct] - m) * p.scale_log2);
#pragma unroll
        for (int c = 0; c < 8; ++c) lds.o[wave][(c * CT + ct) * 64 + lane] = st.o[ct][c] * a;
    }
    if (static_cast<int>(threadIdx.x) < columns) {
        const int c = threadIdx.x;
        float m = lds.m[0][c], l = 0.f;
#pragma unroll
        for (int w = 1; w < kWaves; ++w) m = fmaxf(m, lds.m[w][c]);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) l += lds.l[w][c] * (lds.m[w][c] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((lds.m[w][c] - m) * p.scale_log2));
        part_ml[c * 2] = m * p.scale_log2;
        part_ml[c * 2 + 1] = l;
    }
    __syncthreads();
#pragma unroll
    for (int i = static_cast<int>(threadIdx.x); i < 8 * CT * 64; i += kThreads) {
        const int n = i & 63, ct = (i >> 6) % CT, c = (i >> 6) / CT, column = ct * 16 + (n & 15);
        float4_t v = lds.o[0][i];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) v += lds.o[w][i];
        if (column < columns) *reinterpret_cast<float4_t *>(part_o + column * static_cast<int>(kHeadDim) + c * 16 + (n >> 4) * 4) = v;
    }
}

// A part of a sequence's own rows, by one wave.  new_row: the sequence's length,
// whose new row the wave appends, or -1: one more key behind the part's (fp16
// pages), or the last of the part's keys (8-bit pages).
template <int CODE, bool F32>
__device__ inline void attend_own(const SharedRows &p, const SharedSet &set, int r, uint32_t g, int keys, int first, int end, int new_row, float *part_o,
                                  float *part_ml) {
    const int lane = threadIdx.x & 63, row = lane & 15, kg = lane >> 4;
    SharedQuery<CODE, F32> query[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) query[kb].send(p, set, r, g, kb);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (CODE != PVLC_HIP_KV_F16) {
        if (new_row >= 0) append_q8<CODE, F32>(p, set.first + r, new_row, g);  // uniform
    }
    Attend<CODE, F32, 1> loop;
    loop.begin(pages_of(p, set.first + r, set.shared, keys, g), first, end, 1);
    half8_t qf[1][4];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) query[kb].take(&qf[0][kb], &qf[0][kb + 2]);
    const int limit[1] = {keys};
    AttendState<1> st;
    st.clear();
    loop.run(qf, keys / kAttendStep, limit, keys, p.scale_log2, st);
    if (loop.bad && lane == 0) atomicOr(p.error_word, 2u);
    if constexpr (CODE == PVLC_HIP_KV_F16) {
        if (new_row >= 0) append_and_attend<F32>(p, set.first + r, new_row, g, qf[0], st);  // uniform
    }
    const float l = column_sum(st.l[0]);
    if (row < static_cast<int>(kGroup)) {
        if (kg == 0) {
            part_ml[row * 2] = st.m[0] * p.scale_log2;
            part_ml[row * 2 + 1] = l;
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) *reinterpret_cast<float4_t *>(part_o + row * static_cast<int>(kHeadDim) + c * 16 + kg * 4) = st.o[0][c];
    }
}

// Workgroup: share u and kv head, and a part of the shared rows, or a part of
// every sequence's own ones, a wave each.
template <int CODE, bool F32, int CT>
__global__ __launch_bounds__(kThreads, 2) void shared_attention_kernel(SharedRows p) {
    __shared__ SharedLds<CT> lds;
    constexpr int kNewRow = CODE == PVLC_HIP_KV_F16;  // (not a key of the parts')
    const uint32_t g = blockIdx.x & 1u;
    uint32_t b = blockIdx.x >> 1;
    const bool common = b < p.shares * p.shared_parts;  // uniform, as all below
    if (!common) b -= p.shares * p.shared_parts;
    const uint32_t per = common ? p.shared_parts : p.own_parts, u = b / per;
    const int part = static_cast<int>(b % per);
    SharedSet set;
    if (!find_set<CT>(p, u, &set)) return;
    const int shared_parts = static_cast<int>(p.shared_parts), own_parts = static_cast<int>(p.own_parts);
    const size_t unit = static_cast<size_t>(u) * 2 + g;
    float *const part_o = p.part_o + unit * p.unit_columns * kHeadDim, *const part_ml = p.part_ml + unit * p.unit_columns * 2;
    if (common) {
        const int steps = part_steps(set.shared, shared_parts, kLeastShared), first = part * steps, column = part * CT * 16;
        if (part < parts_of(set.shared, shared_parts, kLeastShared))
            attend_shared<CODE, F32, CT>(p, set, g, first, min(first + steps, (set.shared + kAttendStep - 1) / kAttendStep),
                                         part_o + column * static_cast<int>(kHeadDim), part_ml + column * 2, lds);
        return;
    }
    const int r = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    if (r >= set.count) return;
    const int len = set.len(r), keys = len + 1 - kNewRow - set.shared;
    if (!fits(p, len)) {
        if ((threadIdx.x & 63) == 0 && part == 0) atomicOr(p.error_word, 1u);
        return;
    }
    const int parts = max(parts_of(keys, own_parts, kLeastOwn), kNewRow);
    if (part >= parts) return;
    const int steps = part_steps(keys, own_parts, kLeastOwn), first = part * steps;
    const int column = shared_parts * CT * 16 + (r * own_parts + part) * static_cast<int>(kGroup);
    attend_own<CODE, F32>(p, set, r, g, keys, first, min(first + steps, (keys + kAttendStep - 1) / kAttendStep), part == (kNewRow ? 0 : parts - 1) ? len : -1,
                          part_o + column * static_cast<int>(kHeadDim), part_ml + column * 2);
}

// Workgroup: a sequence and kv head; thread t has head t / 32 and dims t % 32 * 4
// .. + 3.  The parts are loaded with the lengths that say which of them are there.
template <int CODE, bool F32, int CT>
__global__ __launch_bounds__(256) void shared_join_kernel(SharedRows p) {
    constexpr int kNewRow = CODE == PVLC_HIP_KV_F16, kBatch = 16;
    const uint32_t g = blockIdx.x & 1u, u = (blockIdx.x >> 1) / (2 * CT);
    const int r = static_cast<int>((blockIdx.x >> 1) % (2 * CT));
    const int shared_parts = static_cast<int>(p.shared_parts), own_parts = static_cast<int>(p.own_parts), all = shared_parts + own_parts;
    const int head = threadIdx.x >> 5, d0 = (threadIdx.x & 31) * 4;
    const size_t unit = static_cast<size_t>(u) * 2 + g;
    const float *part_o = p.part_o + unit * p.unit_columns * kHeadDim, *part_ml = p.part_ml + unit * p.unit_columns * 2;
    typedef float float2v __attribute__((ext_vector_type(2)));
    float2v ml[kBatch];
    float4_t v[kBatch];
    auto load = [&](int i0) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int part = min(i0 + i, all - 1);
            const int column = (part < shared_parts ? part * CT * 16 + r * static_cast<int>(kGroup)
                                                    : shared_parts * CT * 16 + (r * own_parts + part - shared_parts) * static_cast<int>(kGroup)) + head;
            ml[i] = *reinterpret_cast<const float2v *>(part_ml + column * 2);
            v[i] = *reinterpret_cast<const float4_t *>(part_o + column * static_cast<int>(kHeadDim) + d0);
        }
    };
    load(0);
    __builtin_amdgcn_sched_barrier(0);
    SharedSet set;
    if (!find_set<CT>(p, u, &set) || r >= set.count) return;
    const int len = set.len(r);
    if (!fits(p, len)) return;
    const int shared = parts_of(set.shared, shared_parts, kLeastShared), own = max(parts_of(len + 1 - kNewRow - set.shared, own_parts, kLeastOwn), kNewRow);
    float m = -INFINITY, l = 0.f;
    float4_t o{0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0;;) {
        float top = m;
        auto there = [&](int i) { return i0 + i < shared_parts ? i0 + i < shared : i0 + i - shared_parts < own; };
#pragma unroll
        for (int i = 0; i < kBatch; ++i) top = there(i) ? fmaxf(top, ml[i][0]) : top;
        const float a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
        l *= a;
        o *= a;
        m = top;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (there(i)) {
                const float w = ml[i][0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[i][0] - top);
                l += ml[i][1] * w;
                o += v[i] * w;
            }
        }
        i0 += kBatch;
        if (i0 >= shared_parts + own) break;
        load(i0);
    }
    const float4_t f = o * (1.0f / l);
    const size_t at = (static_cast<size_t>(set.first + r) * kQueryHeads + g * kGroup + head) * kHeadDim + d0;
    if constexpr (F32) *reinterpret_cast<float4_t *>(static_cast<float *>(p.out) + at) = f;
    else *reinterpret_cast<half4_t *>(static_cast<uint16_t *>(p.out) + at) = half4_t{to_h(f[0]), to_h(f[1]), to_h(f[2]), to_h(f[3])};
}

template <int CODE, bool F32, int CT>
void launch(const SharedRows &p, hipStream_t stream) {
    hipLaunchKernelGGL((shared_attention_kernel<CODE, F32, CT>), dim3(2 * p.shares * (p.shared_parts + p.own_parts)), dim3(kThreads), 0, stream, p);
    hipLaunchKernelGGL((shared_join_kernel<CODE, F32, CT>), dim3(2 * p.shares * 2 * CT), dim3(256), 0, stream, p);
}

template <bool F32, int CT>
void launch_code(const SharedRows &p, hipStream_t stream) {
    if (p.code == PVLC_HIP_KV_F16) launch<PVLC_HIP_KV_F16, F32, CT>(p, stream);
    else if (p.code == PVLC_HIP_KV_E4M3) launch<PVLC_HIP_KV_E4M3, F32, CT>(p, stream);
    else launch<PVLC_HIP_KV_INT8, F32, CT>(p, stream);
}

}  // namespace

int launch_shared_decode(const SharedRows &rows, void *stream) {
    SharedRows p = rows;
    p.scale_log2 = kAttendLog2e / sqrtf(static_cast<float>(kHeadDim));
    const auto st = static_cast<hipStream_t>(stream);
    if (p.columns == 1) p.f32 ? launch_code<true, 1>(p, st) : launch_code<false, 1>(p, st);
    else p.f32 ? launch_code<true, 2>(p, st) : launch_code<false, 2>(p, st);
    return static_cast<int>(hipGetLastError());
}

}  // namespace pvlc
