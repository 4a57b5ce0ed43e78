// Rows of several sequences into the pages behind what each holds, keys
// rotated on the way; fp16 or 8-bit pages.

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "pvlc_q8.hpp"
#include "packed_plan.hpp"
#include "ragged_device.hpp"

namespace pvlc {
namespace {

constexpr int kThreads = 256;
constexpr int kPad = 8;  // elements behind each LDS row of 256 dims, against bank conflicts
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
constexpr uint32_t kLargestHalf = 0x7BFF;  // 65504; infinity is the next, NaN behind

__device__ inline uint32_t largest(u16x8_t x) {
    uint16_t m = x[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) m = max(m, x[j]);
    return m;
}
// Over the row of 16 lanes.
__device__ inline uint32_t row_max(uint32_t x) {
#define PVLC_ROW_MAX(CTRL) x = max(x, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, 0xF, 0xF, false)))
    PVLC_ROW_MAX(0xB1);
    PVLC_ROW_MAX(0x4E);
    PVLC_ROW_MAX(0x124);
    PVLC_ROW_MAX(0x128);
#undef PVLC_ROW_MAX
    return x;
}

// A workgroup for each 16-token block that a sequence writes to, both heads.
// Keys: every thread rotates one pair of 8-dim chunks, c and c + 8, which are
// each other's partners (item = head, pair, token).  fp16 pages: 16 threads fill
// a 256-byte run of the key slab, and the values are turned through LDS into
// 32-byte rows of the value slab.  8-bit pages: the block's exponents come from
// the sizes, and rows that the block holds already are rounded again where these
// grew; 8 dims of a token are 8 bytes, stored from the registers (a wave's fill
// runs of 64 bytes; with the keys in LDS too, as they had been, a compute unit held
// six workgroups in place of eight).  Other tokens of a block stay as they are.
//
// Short calls are bound by the chain of dependent rounds: the sequence; its
// table entry, positions and rows; cos and sin; (8 bits: the old block with the
// rows); the stores.  A few rows for each of 24 sequences 4.4 us a call, a page of 1157
// f32 rows into e4m3 4.4.  Long calls: 16 prompts of 90 to 2010 fp16 rows (20 MB) 7.4
// us, 2.8 TB/s with the launch; 8 documents of 4096 to 14336 rows into int8 (100 MB)
// 25.1 us, 4.0 TB/s of a copy's 5.1: sizes and codes are 60% of their vector
// instructions.
template <bool F32, int CODE>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(AppendRows p) {
    constexpr bool kQ8 = CODE != PVLC_HIP_KV_F16;
    __shared__ __align__(16) uint16_t sv[kBlockTokens][kRowElems + kPad];
    __shared__ uint32_t sm_size[2][kKvHeads], sm_special;
    typedef std::conditional_t<F32, float, uint16_t> Element;
    typedef std::conditional_t<F32, float4_t, half8_t> Raw;
    constexpr int kLoads = F32 ? 2 : 1, kElems = F32 ? 4 : 8;
    const int i = threadIdx.x;
    uint32_t share = blockIdx.x;
    if constexpr (!kQ8) {
        // A plan for the launch behind this one, by one workgroup more.
        if (p.plan.items) {
            if (share == 0) {
                make_packed_plan(p.ragged, p.plan);
                return;
            }
            --share;
        }
    }
    const SeqRows q = find_share<16, 2>(p.ragged, share);
    if ((!q.ok || q.told) && i == 0 && p.error_word) atomicOr(p.error_word, 1u);
    if (!q.ok) return;  // uniform, as below
    const int64_t end = static_cast<int64_t>(q.held) + q.count;
    const int64_t block = static_cast<int64_t>(q.held / static_cast<int>(kBlockTokens)) + q.share;
    if (q.count == 0 || block * kBlockTokens >= end) return;
    // Tokens [lo, hi) of the block are the call's; row r of the call is token base + r of the block.
    const int lo = static_cast<int>(max(q.held - block * kBlockTokens, static_cast<int64_t>(0)));
    const int hi = static_cast<int>(min(end - block * kBlockTokens, static_cast<int64_t>(kBlockTokens)));
    const int64_t row0 = q.begin + (block * kBlockTokens - q.held);  // of the block's first token
    const int64_t entry = static_cast<int64_t>(q.seq) * p.ragged.max_blocks + block;
    const Element *keys = static_cast<const Element *>(p.key), *values = static_cast<const Element *>(p.value);

    const int tt = i & 15, c = (i >> 4) & 7, hh = i >> 7;
    const int64_t t = row0 + min(max(tt, lo), hi - 1);  // (tokens that are not the call's repeat one that is)
    // (Arrays that are not given are read through the key pointer, so that no load waits behind a branch.)
    const int32_t *stand_in = static_cast<const int32_t *>(p.key);
    const int32_t id_given = load_const(p.ragged.tables ? p.ragged.tables + entry : stand_in, 0);
    const int32_t pos_given = *(p.positions ? p.positions + t : stand_in);
    Raw key[2][kLoads], val[2][kLoads];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int k = i + r * kThreads;
        const Element *ks = keys + t * p.key_stride + hh * kHeadDim + c * 8 + r * 64;
        const Element *vs = values + (row0 + min(max(k >> 5, lo), hi - 1)) * p.value_stride + (k & 31) * 8;
#pragma unroll
        for (int f = 0; f < kLoads; ++f) {
            key[r][f] = *reinterpret_cast<const Raw *>(ks + f * kElems);
            val[r][f] = *reinterpret_cast<const Raw *>(vs + f * kElems);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    const int64_t pos = p.positions ? pos_given : t - q.begin + q.held;
    const bool rope = p.rope_cos != nullptr && pos >= 0 && pos < static_cast<int64_t>(p.rope_rows);
    float4_t cs[2], sn[2];
    {
        const float *cr = rope ? p.rope_cos + pos * 64 + c * 8 : reinterpret_cast<const float *>(stand_in);
        const float *sr = rope ? p.rope_sin + pos * 64 + c * 8 : reinterpret_cast<const float *>(stand_in);
#pragma unroll
        for (int f = 0; f < 2; ++f) {
            cs[f] = *reinterpret_cast<const float4_t *>(cr + f * 4);
            sn[f] = *reinterpret_cast<const float4_t *>(sr + f * 4);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    bool ok;
    const uint32_t id = checked_block(p.ragged, p.ragged.tables ? id_given : entry, &ok);  // uniform
    u32x2_t old_k[2]{};
    q8x4_t old_v{};
    uint32_t old_e = 0;
    const bool whole = lo == 0 && hi == static_cast<int>(kBlockTokens);  // uniform
    // 8 bits: the bytes of dims c * 8 .. of token tt (64 dims on: 256 bytes on), and (head, dim) i of the values.
    const size_t slab = static_cast<size_t>(id) * kKvHeads * kQ8SlabBytes;
    uint8_t *const key_bytes = static_cast<uint8_t *>(p.key_cache) + slab + hh * static_cast<int>(kQ8SlabBytes) + (tt >> 2) * 512 + (c >> 1) * 64 + (tt & 3) * 16 + (c & 1) * 8;
    uint8_t *const value_bytes = static_cast<uint8_t *>(p.value_cache) + slab + i * 16;
    if (kQ8 && ok && !whole) {
#pragma unroll
        for (int r = 0; r < 2; ++r) old_k[r] = *reinterpret_cast<const u32x2_t *>(key_bytes + r * 256);
        old_v = *reinterpret_cast<const q8x4_t *>(value_bytes);
        old_e = *reinterpret_cast<const uint16_t *>(p.exponents + (static_cast<size_t>(id) * kKvHeads + hh) * 2);
    }
    if (kQ8 && i < 2 * static_cast<int>(kKvHeads)) sm_size[i >> 1][i & 1] = 0;
    if (kQ8 && i == 0) sm_special = 0;
    half8_t out[2];
    if (__any(rope)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {  // as rotate_chunk rotates
            const float x = static_cast<float>(key[0][j / kElems][j % kElems]);
            const float y = static_cast<float>(key[1][j / kElems][j % kElems]);
            const float co = cs[j >> 2][j & 3], si = sn[j >> 2][j & 3];
            out[0][j] = to_h(x * co + (-y) * si);
            out[1][j] = to_h(y * co + x * si);
        }
    }
    if (__any(!rope) && !rope) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            if constexpr (F32) {
#pragma unroll
                for (int j = 0; j < 8; ++j) out[r][j] = to_h(key[r][j / kElems][j % kElems]);
            } else {
                out[r] = key[r][0];  // as given, bit for bit
            }
        }
    }
    half8_t v[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        if constexpr (F32) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[r][j] = to_h(val[r][j / kElems][j % kElems]);
        } else {
            v[r] = val[r][0];
        }
        const int k = i + r * kThreads;
        *reinterpret_cast<half8_t *>(&sv[k >> 5][(k & 31) * 8]) = v[r];
    }
    if (p.error_word) {
        if (!ok && i == 0) atomicOr(p.error_word, 2u);
        if (!rope && p.rope_cos != nullptr && c == 0 && hh == 0 && tt >= lo && tt < hi) atomicOr(p.error_word, 4u);
    }
    if constexpr (!kQ8) {
        if (p.odd) {  // for the packed prompts: which blocks have values that are not finite (a byte for each wave)
            const u16x8_t every = static_cast<uint16_t>(0x7FFF);
            const u16x8_t size = __builtin_elementwise_max(__builtin_bit_cast(u16x8_t, v[0]) & every, __builtin_bit_cast(u16x8_t, v[1]) & every);
            const bool odd = __any(largest(size) > kLargestHalf) != 0;
            if ((i & 63) == 0) reinterpret_cast<uint8_t *>(p.odd + share)[i >> 6] = odd;
        }
        if (ok && tt >= lo && tt < hi) {
            uint16_t *dst = static_cast<uint16_t *>(p.key_cache) + (static_cast<size_t>(id) * kKvHeads + hh) * kBlockHeadElems + c * 128 + key_slot(tt) * 8;
            *reinterpret_cast<half8_t *>(dst) = out[0];
            *reinterpret_cast<half8_t *>(dst + 8 * 128) = out[1];
        }
        __syncthreads();
        if (!ok) return;
        uint16_t *dst = static_cast<uint16_t *>(p.value_cache) + static_cast<size_t>(id) * kKvHeads * kBlockHeadElems + i * kBlockTokens;  // (head, dim) i
        if (whole) {
            u16x8_t a, b;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                a[e] = sv[e][i];
                b[e] = sv[e + 8][i];
            }
            *reinterpret_cast<u16x8_t *>(dst) = a;
            *reinterpret_cast<u16x8_t *>(dst + 8) = b;
        } else {
            for (int e = lo; e < hi; ++e) dst[e] = sv[e][i];
        }
    } else {
        __syncthreads();  // the rows are in LDS, and sm_size is cleared
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            // A wave's key items are of one head; 16 lanes hold the values of one
            // head.  fp16 sizes are in the order of their bits.
            const u16x8_t every = static_cast<uint16_t>(0x7FFF);
            const u16x8_t a = __builtin_bit_cast(u16x8_t, w ? v[0] : out[0]) & every, b = __builtin_bit_cast(u16x8_t, w ? v[1] : out[1]) & every;
            uint32_t size = largest(__builtin_elementwise_max(a, b));
            if (size > kLargestHalf) {  // an infinity counts as the largest value, a NaN as none
                size = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (a[j] <= kLargestHalf + 1u) size = max(size, min(static_cast<uint32_t>(a[j]), kLargestHalf));
                    if (b[j] <= kLargestHalf + 1u) size = max(size, min(static_cast<uint32_t>(b[j]), kLargestHalf));
                }
                sm_special = 1;
            }
            size = row_max(size);
            if ((i & 15) == 0) atomicMax(&sm_size[w][w ? (i >> 4) & 1 : hh], size);
        }
        __syncthreads();
        if (!ok) return;
        const bool special = sm_special != 0;  // uniform
        // Four fp16 values to codes.  Without infinities and NaN nothing is clamped, and the sum of
        // an int8 code and 1.5 2^23 has the code, rounded to even, as its low byte.
        auto encode = [&](_Float16 x0, _Float16 x1, _Float16 x2, _Float16 x3, float inv) -> uint32_t {
            const float f0 = static_cast<float>(x0), f1 = static_cast<float>(x1), f2 = static_cast<float>(x2), f3 = static_cast<float>(x3);
            if (special) return q8_encode<CODE>(q8_value(f0) * inv, q8_value(f1) * inv, q8_value(f2) * inv, q8_value(f3) * inv);
            if constexpr (CODE == PVLC_HIP_KV_E4M3) {
                return q8_encode<CODE>(f0 * inv, f1 * inv, f2 * inv, f3 * inv);
            } else {
                constexpr float kWhole = 12582912.0f;
                auto bits = [&](float f) { return __float_as_uint(__builtin_fmaf(f, inv, kWhole)); };
                return __builtin_amdgcn_perm(bits(f1), bits(f0), 0x0C0C0400u) | __builtin_amdgcn_perm(bits(f3), bits(f2), 0x04000C0Cu);
            }
        };
        int e[2], grown[2];  // of head hh: the thread's keys and its row of the values
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            e[w] = q8_exponent<CODE>(static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(sm_size[w][hh]))));
            const int before = static_cast<int>((old_e >> (8 * w)) & 255) - kQ8Bias;
            if (lo > 0) e[w] = max(e[w], before);
            grown[w] = lo > 0 ? e[w] - before : 0;
        }
        if (tt < hi && (tt >= lo || grown[0] > 0)) {
            const float inv = exp2_whole(-e[0]);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const half8_t &x = out[r];
                u32x2_t codes = {encode(x[0], x[1], x[2], x[3], inv), encode(x[4], x[5], x[6], x[7], inv)};
                if (lo > 0) {  // uniform
#pragma unroll
                    for (int w = 0; w < 2; ++w) codes[w] = tt < lo ? q8_requantise<CODE>(old_k[r][w], grown[0]) : codes[w];
                }
                *reinterpret_cast<u32x2_t *>(key_bytes + r * 256) = codes;
            }
        }
        {
            const float inv = exp2_whole(-e[1]);
            q8x4_t codes;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                auto value = [&](int j) { return __builtin_bit_cast(_Float16, sv[w * 4 + j][i]); };
                codes[w] = encode(value(0), value(1), value(2), value(3), inv);
            }
            if (!whole) {
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint32_t again = grown[1] > 0 ? q8_requantise<CODE>(old_v[w], grown[1]) : old_v[w];
                    uint32_t x = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int token = w * 4 + j;
                        x |= (token < lo ? again : token < hi ? codes[w] : old_v[w]) & (0xFFu << (8 * j));
                    }
                    codes[w] = x;
                }
            }
            *reinterpret_cast<q8x4_t *>(value_bytes) = codes;
        }
        if ((i & 127) == 0)
            *reinterpret_cast<uint16_t *>(p.exponents + (static_cast<size_t>(id) * kKvHeads + hh) * 2) =
                static_cast<uint16_t>((e[0] + kQ8Bias) | (e[1] + kQ8Bias) << 8);
    }
}

template <bool F32>
void (*append_kernel(uint32_t code))(AppendRows) {
    return code == PVLC_HIP_KV_F16 ? kv_append_kernel<F32, PVLC_HIP_KV_F16>
           : code == PVLC_HIP_KV_E4M3 ? kv_append_kernel<F32, PVLC_HIP_KV_E4M3>
                                      : kv_append_kernel<F32, PVLC_HIP_KV_INT8>;
}

}  // namespace

int launch_kv_append(const AppendRows &p, void *stream) {
    const RaggedRows &r = p.ragged;
    const uint32_t shares = r.offsets ? r.rows / kBlockTokens + 2 * r.num_seqs : r.num_seqs * shares_of_each<kBlockTokens, 2>(r.each);
    hipLaunchKernelGGL(p.f32 ? append_kernel<true>(p.code) : append_kernel<false>(p.code), dim3(shares + (p.plan.items ? 1 : 0)), dim3(kThreads), 0,
                       static_cast<hipStream_t>(stream), p);
    return static_cast<int>(hipGetLastError());
}

}  // namespace pvlc
