// Attention of a few columns of 16 queries over paged keys and values, by one
// wave: the loop of the shared decode and of small packed prompts.
//
//   S^T[key][query] = K Q^T        v_mfma_f32_16x16x32_f16
//   O^T[dim][query] += V^T P^T     the same (8-bit pages: ..._bf16)
//
// A step is 32 keys, two cache tiles.  The rows of score MFMA h are given to the
// keys such that lane (query, kg) receives keys kg * 8 + h * 4 + r: 8 consecutive
// ones after both, which is its operand of the second product.  With the values
// as the first operand a lane keeps one query's outputs, so the softmax's
// factors never leave the lane.  Keys and values come from the pages into
// registers, whole lines a load, a step ahead of their use: where few queries read
// each key, LDS would only add a round.
//
// Sums and outputs are f32.  Scores are products of fp16 (8-bit codes are exact in
// it).  Weights are fp16, with f32 operands pairs of it (22 bits); over 8-bit pages,
// whose powers of two they carry, two or three bf16 terms (16 and 24 bits).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "pvlc_q8.hpp"
#include "ragged_device.hpp"

namespace pvlc {

constexpr int kAttendStep = 32;
constexpr float kAttendLog2e = 1.4426950408889634f;
constexpr float kAttendRescaleLog2 = 8.0f;  // the softmax reference moves only past 2^8

// The pages of one sequence and kv head.
struct AttendPages {
    const uint8_t *keys, *values, *exponents;
    const int32_t *table;  // the sequence's row, or null: blocks first, first + 1, ..
    uint32_t first, num_blocks, head;
    int last_tile;  // tiles behind it are read as it
};

// A block outside the planes is read as block 0, and `bad` set, for the wave.
__device__ inline uint32_t attend_block(const AttendPages &p, int tile, bool *bad) {
    const int64_t id = p.table ? p.table[tile] : static_cast<int64_t>(p.first) + tile;
    const bool out = id < 0 || id >= static_cast<int64_t>(p.num_blocks);
    *bad |= __any(out) != 0;
    return out ? 0u : static_cast<uint32_t>(id);
}

// First dim of the 8 that a lane's operand kb of a score MFMA covers.  8-bit keys
// come as 16 dims a load, two operands.  Operands kb and kb + 2 rotate together.
template <int CODE>
__device__ constexpr int attend_dim(int kb, int kg) {
    return CODE == PVLC_HIP_KV_F16 ? kb * 32 + kg * 8 : (kb >> 1) * 64 + kg * 16 + (kb & 1) * 8;
}

// Eight rotated (exactly as rotate_chunk does) dims and their partners.
template <bool F32>
struct AttendQuery {
    typedef std::conditional_t<F32, float4_t, half8_t> Raw;
    typedef std::conditional_t<F32, float, uint16_t> Element;
    static constexpr int kLoads = F32 ? 2 : 1, kElems = F32 ? 4 : 8;
    Raw x[2][kLoads];
    __device__ void load(const Element *row, int d0) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int f = 0; f < kLoads; ++f) x[k][f] = *reinterpret_cast<const Raw *>(row + d0 + k * 64 + f * kElems);
    }
    __device__ void rotate(bool rope, const float4_t (&cs)[2], const float4_t (&sn)[2], half8_t *lo, half8_t *hi) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float c = cs[j >> 2][j & 3], s = sn[j >> 2][j & 3];
            const float a = static_cast<float>(x[0][j / kElems][j % kElems]), b = static_cast<float>(x[1][j / kElems][j % kElems]);
            (*lo)[j] = to_h(rope ? a * c + (-b) * s : a);
            (*hi)[j] = to_h(rope ? b * c + a * s : b);
        }
    }
};

// Softmax state of CT columns: O^T (dims c * 16 + kg * 4 + r of the lane's query),
// the reference and the lane's own part of the sum.
template <int CT>
struct AttendState {
    float4_t o[CT][8];
    float m[CT], l[CT];
    __device__ void clear() {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
            for (int c = 0; c < 8; ++c) o[ct][c] = float4_t{0.f, 0.f, 0.f, 0.f};
            m[ct] = -INFINITY;
            l[ct] = 0.f;
        }
    }
};

// Over the 4 lanes of a query (l, l ^ 16, l ^ 32, l ^ 48).
typedef uint32_t attend_u32x2 __attribute__((ext_vector_type(2)));
__device__ inline float column_max(float c) {
    attend_u32x2 v = __builtin_amdgcn_permlane16_swap(__float_as_uint(c), __float_as_uint(c), false, false);
    c = fmaxf(__uint_as_float(v[0]), __uint_as_float(v[1]));
    v = __builtin_amdgcn_permlane32_swap(__float_as_uint(c), __float_as_uint(c), false, false);
    return fmaxf(__uint_as_float(v[0]), __uint_as_float(v[1]));
}
__device__ inline float column_sum(float c) {
    attend_u32x2 v = __builtin_amdgcn_permlane16_swap(__float_as_uint(c), __float_as_uint(c), false, false);
    c = __uint_as_float(v[0]) + __uint_as_float(v[1]);
    v = __builtin_amdgcn_permlane32_swap(__float_as_uint(c), __float_as_uint(c), false, false);
    return __uint_as_float(v[0]) + __uint_as_float(v[1]);
}

// Infinities and NaN among values become 0.  (A weight of 0, for a key that a query
// does not see, would make them NaN.)
__device__ inline bool is_odd(uint16_t v) { return (v & 0x7C00) == 0x7C00; }
__device__ inline void clean(half8_t &v) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const _Float16 x = v[e];  // (a bit cast of the element itself takes the first one's bits)
        v[e] = is_odd(__builtin_bit_cast(uint16_t, x)) ? static_cast<_Float16>(0.0f) : x;
    }
}
// Such a value, where the query sees its key; else 0.
__device__ inline float odd_value(uint16_t v, bool seen) { return seen && is_odd(v) ? static_cast<float>(__builtin_bit_cast(_Float16, v)) : 0.f; }

// Keys and values of a step as they lie in the pages.
template <int CODE>
struct AttendTile {
    static constexpr bool kQ8 = CODE != PVLC_HIP_KV_F16;
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    typedef std::conditional_t<kQ8, q8x4_t, half8_t> Key;
    typedef std::conditional_t<kQ8, u32x2, half8_t> Value;
    Key k[2][kQ8 ? 2 : 4];
    Value v[8];
    uint32_t ek, ev;  // 8 bits: exponents of the tile of this lane's keys

    __device__ void load_k(const AttendPages &p, uint32_t b0, uint32_t b1, int row, int kg) {
        const size_t slab = static_cast<size_t>(row < 8 ? b0 : b1) * kKvHeads + p.head;
        if constexpr (kQ8) {
            // row 4 a + t of MFMA h is token t of quad 2 (a & 1) + h of tile a >> 1
            const uint8_t *src = p.keys + slab * kQ8SlabBytes + ((row >> 2) & 1) * 1024 + (row & 3) * 16 + kg * 64;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int c = 0; c < 2; ++c) k[h][c] = *reinterpret_cast<const q8x4_t *>(src + h * 512 + c * 256);
            ek = p.exponents[(static_cast<size_t>(kg < 2 ? b0 : b1) * kKvHeads + p.head) * 2];
        } else {
            const uint16_t *src = reinterpret_cast<const uint16_t *>(p.keys) + slab * kBlockHeadElems;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int kb = 0; kb < 4; ++kb)
                    k[h][kb] = *reinterpret_cast<const half8_t *>(src + (kb * 4 + kg) * 128 + (h * 8 + (row & 7)) * 8);
        }
    }
    __device__ void load_v(const AttendPages &p, uint32_t b0, uint32_t b1, int row, int kg) {
        const size_t slab = static_cast<size_t>(kg < 2 ? b0 : b1) * kKvHeads + p.head;
        if constexpr (kQ8) {
#pragma unroll
            for (int c = 0; c < 8; ++c)
                v[c] = *reinterpret_cast<const u32x2 *>(p.values + slab * kQ8SlabBytes + (c * 16 + row) * 16 + (kg & 1) * 8);
            ev = p.exponents[slab * 2 + 1];
        } else {
            const uint16_t *src = reinterpret_cast<const uint16_t *>(p.values) + slab * kBlockHeadElems;
#pragma unroll
            for (int c = 0; c < 8; ++c) v[c] = *reinterpret_cast<const half8_t *>(src + (c * 16 + row) * 16 + (kg & 1) * 8);
        }
    }
    __device__ half8_t key(int h, int kb) const {
        if constexpr (kQ8) return q8_half8<CODE>(k[h][kb >> 1][(kb & 1) * 2], k[h][kb >> 1][(kb & 1) * 2 + 1]);
        else return k[h][kb];
    }
    // Values of keys key .. key + 7 that lie at `valid` or behind become 0: what
    // the pages hold there may be NaN, and a weight of 0 would not remove it.
    __device__ void keep(int key, int valid) {
        typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
        if constexpr (kQ8) {
            const int n = min(max(valid - key, 0), 8);
            const uint64_t mask = n == 8 ? ~0ull : (1ull << (8 * n)) - 1;
            const u32x2 m = __builtin_bit_cast(u32x2, mask);
#pragma unroll
            for (int c = 0; c < 8; ++c) v[c] &= m;
        } else {
            u32x4 m;
#pragma unroll
            for (int d = 0; d < 4; ++d) m[d] = key + 2 * d + 1 < valid ? ~0u : key + 2 * d < valid ? 0xffffu : 0u;
#pragma unroll
            for (int c = 0; c < 8; ++c) v[c] = __builtin_bit_cast(half8_t, __builtin_bit_cast(u32x4, v[c]) & m);
        }
    }
};

// Steps first, first + stride, .. below end of a sequence's keys.  A column's
// query sees the keys below its limit; steps below `masked` lie below every
// limit.  `valid` keys are the sequence's (see AttendTile::keep).  begin() sends
// out the first step's loads, so that the queries can be made ready under them.
// CLEAN: limits differ, and if `odd`, values that are not finite are left out of
// the masked steps; add_odd adds them where they are seen.
template <int CODE, bool F32, int CT, bool CLEAN = false>
struct Attend {
    bool odd = false;  // uniform
    bool bad = false;  // uniform: a block of the steps, or of the next 32, lies outside the planes
    AttendPages p;
    int first, end, stride;
    uint32_t ids;  // blocks, one per lane: lane 2 i + j holds tile j of step i0 + i (32 steps a load)
    AttendTile<CODE> tile;

    __device__ int tile_of(int i0) const {
        const int lane = threadIdx.x & 63;
        return min(2 * (first + (i0 + (lane >> 1)) * stride) + (lane & 1), p.last_tile);
    }
    __device__ uint32_t id_of(int i, int j) const {
        return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(ids), 2 * (i & 31) + j));
    }
    __device__ __attribute__((always_inline)) void begin(const AttendPages &pages, int from, int to, int by) {
        p = pages;
        first = from;
        end = to;
        stride = by;
        if (first >= end) return;  // uniform
        const int lane = threadIdx.x & 63, row = lane & 15, kg = lane >> 4;
        ids = attend_block(p, tile_of(0), &bad);
        tile.load_k(p, id_of(0, 0), id_of(0, 1), row, kg);
        tile.load_v(p, id_of(0, 0), id_of(0, 1), row, kg);
        __builtin_amdgcn_sched_barrier(0);
    }
    __device__ __attribute__((always_inline)) void run(const half8_t (&qf)[CT][4], int masked, const int (&limit)[CT], int valid, float scale,
                                                       AttendState<CT> &st);
    __device__ void add_odd(int masked, const int (&limit)[CT], int valid, AttendState<CT> &st) const {
        const int kg = (threadIdx.x & 63) >> 4;
#pragma unroll 1
        for (int s = first; s < end; s += stride) {
            if (s < masked) continue;
#pragma unroll 1
            for (int key = s * kAttendStep; key < min((s + 1) * kAttendStep, valid) && key / static_cast<int>(kBlockTokens) <= p.last_tile; ++key) {
                bool seen = false;  // (by the loop)
                const size_t slab = static_cast<size_t>(attend_block(p, key / static_cast<int>(kBlockTokens), &seen)) * kKvHeads + p.head;
                const uint16_t *src = reinterpret_cast<const uint16_t *>(p.values) + slab * kBlockHeadElems + key % static_cast<int>(kBlockTokens);
#pragma unroll
                for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        __builtin_amdgcn_sched_barrier(0);  // (few loads at once: this is seldom run, and must not cost the loop registers)
#pragma unroll
                        for (int r = 0; r < 4; ++r) st.o[ct][c][r] += odd_value(src[(c * 16 + kg * 4 + r) * static_cast<int>(kBlockTokens)], key < limit[ct]);
                    }
            }
        }
    }
};

template <int CODE, bool F32, int CT, bool CLEAN>
__device__ __attribute__((always_inline)) inline void Attend<CODE, F32, CT, CLEAN>::run(const half8_t (&qf)[CT][4], int masked, const int (&limit)[CT],
                                                                                         int valid, float scale, AttendState<CT> &st) {
    static_assert(!CLEAN || CODE == PVLC_HIP_KV_F16);
    constexpr bool kQ8 = CODE != PVLC_HIP_KV_F16;
    if (first >= end) return;  // uniform
    const int lane = threadIdx.x & 63, row = lane & 15, kg = lane >> 4;
    uint32_t next_ids = 0;

    auto step = [&](auto mask, int s, int i) __attribute__((always_inline)) {
        if ((i & 31) == 0 && s + 32 * stride < end) next_ids = attend_block(p, tile_of(i + 32), &bad);
        float x[CT][8];
        {
            float4_t acc[CT][2];
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                for (int h = 0; h < 2; ++h) acc[ct][h] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kb = 0; kb < 4; ++kb) {
                const half8_t k0 = tile.key(0, kb), k1 = tile.key(1, kb);
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
                    acc[ct][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qf[ct][kb], acc[ct][0], 0, 0, 0);
                    acc[ct][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qf[ct][kb], acc[ct][1], 0, 0, 0);
                }
            }
            const float power = kQ8 ? exp2_whole(static_cast<int>(tile.ek) - kQ8Bias) : 1.f;
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int r = 0; r < 4; ++r) x[ct][h * 4 + r] = kQ8 ? acc[ct][h][r] * power : acc[ct][h][r];
        }
        __builtin_amdgcn_sched_barrier(0);
        // The next step's keys.  (Loads behind the last step would be waited for
        // where the results are joined: a part of one step a wave 1 us longer.)
        if (((i + 1) & 31) == 0) ids = next_ids;
        const uint32_t b0 = id_of(i + 1, 0), b1 = id_of(i + 1, 1);
        const bool more = s + stride < end;  // uniform
        if (more) tile.load_k(p, b0, b1, row, kg);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (mask) {
            const int key = s * kAttendStep + kg * 8;
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) x[ct][e] = key + e < limit[ct] ? x[ct][e] : -INFINITY;
            if ((s + 1) * kAttendStep > valid) tile.keep(key, valid);  // uniform
            if constexpr (CLEAN) {
                if (odd) {
#pragma unroll
                    for (int c = 0; c < 8; ++c) clean(tile.v[c]);
                }
            }
        }
        bool far = false;
        float m_new[CT];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            float c = st.m[ct];
#pragma unroll
            for (int e = 0; e < 8; ++e) c = fmaxf(c, x[ct][e]);
            m_new[ct] = column_max(c);
            far |= (m_new[ct] - st.m[ct]) * scale > kAttendRescaleLog2;
        }
        if (__any(far)) {  // uniform
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                // (a column without a key so far has nothing to rescale)
                const float a = m_new[ct] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((st.m[ct] - m_new[ct]) * scale);
                st.m[ct] = m_new[ct];
                st.l[ct] *= a;
#pragma unroll
                for (int c = 0; c < 8; ++c) st.o[ct][c] *= a;
            }
        }
        if constexpr (!kQ8) {
            // Weights in fp16; with f32 operands as the pair hi = fp16(w), lo =
            // fp16(w - hi), about 22 bits.  The sum takes them as rounded.
            half8_t hi[CT], lo[CT];
            const half2_t ones = {static_cast<_Float16>(1.0f), static_cast<_Float16>(1.0f)};
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                const float ms = st.m[ct] == -INFINITY ? 0.f : st.m[ct] * scale;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(x[ct][e], scale, -ms));
                    hi[ct][e] = to_h(w);
                    if constexpr (F32) lo[ct][e] = to_h(w - static_cast<float>(hi[ct][e]));
                }
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    st.l[ct] = __builtin_amdgcn_fdot2(half2_t{hi[ct][e], hi[ct][e + 1]}, ones, st.l[ct], false);
                    if constexpr (F32) st.l[ct] = __builtin_amdgcn_fdot2(half2_t{lo[ct][e], lo[ct][e + 1]}, ones, st.l[ct], false);
                }
            }
#pragma unroll
            for (int c = 0; c < 8; ++c)
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
                    st.o[ct][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(tile.v[c], hi[ct], st.o[ct][c], 0, 0, 0);
                    if constexpr (F32) st.o[ct][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(tile.v[c], lo[ct], st.o[ct][c], 0, 0, 0);
                }
        } else {
            // The values' power goes to the weights, in bf16 terms (f32's range):
            // two, 16 bits; with f32 operands three.
            constexpr int kTerms = F32 ? 3 : 2;
            bf16x8_t w[kTerms][CT];
            const float power = exp2_whole(static_cast<int>(tile.ev) - kQ8Bias);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                const float ms = st.m[ct] == -INFINITY ? 0.f : st.m[ct] * scale;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[ct][e], scale, -ms));
                    st.l[ct] += x1;
                    float rest = x1 * power;
#pragma unroll
                    for (int t = 0; t < kTerms; ++t) {
                        w[t][ct][e] = static_cast<__bf16>(rest);
                        rest -= static_cast<float>(w[t][ct][e]);
                    }
                }
            }
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const bf16x8_t v = q8_bf16x8<CODE>(tile.v[c][0], tile.v[c][1]);
#pragma unroll
                for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                    for (int t = 0; t < kTerms; ++t) st.o[ct][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, w[t][ct], st.o[ct][c], 0, 0, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        if (more) tile.load_v(p, b0, b1, row, kg);
        __builtin_amdgcn_sched_barrier(0);
    };
    const std::integral_constant<bool, true> yes;
    const std::integral_constant<bool, false> no;
    int s = first, i = 0;
    for (; s < min(end, masked); s += stride, ++i) step(no, s, i);
    for (; s < end; s += stride, ++i) step(yes, s, i);
}

}  // namespace pvlc
