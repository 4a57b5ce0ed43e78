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
// Key piece i (16 bytes) of a block's two 8-bit slabs: its token, and its first dim among both heads.
__device__ inline int q8_key_token(int i) { return ((i >> 5) & 3) * 4 + (i & 3); }
__device__ inline int q8_key_dim(int i) { return (i >> 7) * kHeadDim + ((i >> 2) & 7) * 16; }

// A workgroup for each 16-token block that a sequence writes to, both heads.
// Keys: every thread rotates one pair of 8-dim chunks, c and c + 8, which are
// each other's partners (item = head, pair, token).  fp16 pages: 16 threads fill
// a 256-byte run of the key slab, and the values are turned through LDS into
// 32-byte rows of the value slab.  8-bit pages: both go through LDS, the block's
// exponents come from the sizes, and rows that the block holds already are
// rounded again where these grew.  Other tokens of a block stay as they are.
//
// Short calls are bound by the chain of dependent rounds: the sequence; its
// table entry, positions and rows; cos and sin; (8 bits: the old block with the
// rows); the stores.
template <bool F32, int CODE>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(AppendRows p) {
    constexpr bool kQ8 = CODE != PVLC_HIP_KV_F16;
    __shared__ __align__(16) uint16_t sr[kQ8 ? 2 : 1][kBlockTokens][kRowElems + kPad];
    __shared__ uint32_t sm_size[2][kKvHeads];
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
    if (!q.ok) {
        if (i == 0 && p.error_word) atomicOr(p.error_word, 1u);
        return;  // uniform, as below
    }
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
    const int64_t id_raw = p.ragged.tables ? p.ragged.tables[entry] : entry;
    const int64_t pos = p.positions ? p.positions[t] : t - q.begin + q.held;
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
    const bool rope = p.rope_cos != nullptr && pos >= 0 && pos < static_cast<int64_t>(p.rope_rows);
    float4_t cs[2]{}, sn[2]{};
    if (rope) {
#pragma unroll
        for (int f = 0; f < 2; ++f) {
            cs[f] = *reinterpret_cast<const float4_t *>(p.rope_cos + pos * 64 + c * 8 + f * 4);
            sn[f] = *reinterpret_cast<const float4_t *>(p.rope_sin + pos * 64 + c * 8 + f * 4);
        }
    }
    bool ok;
    const uint32_t id = checked_block(p.ragged, id_raw, &ok);  // uniform
    q8x4_t old_k{}, old_v{};
    uint32_t old_e = 0;
    const bool whole = lo == 0 && hi == static_cast<int>(kBlockTokens);  // uniform
    const size_t slab = static_cast<size_t>(id) * kKvHeads * kQ8SlabBytes + static_cast<size_t>(i) * 16;
    if (kQ8 && ok && !whole) {
        old_k = *reinterpret_cast<const q8x4_t *>(static_cast<uint8_t *>(p.key_cache) + slab);
        old_v = *reinterpret_cast<const q8x4_t *>(static_cast<uint8_t *>(p.value_cache) + slab);
        old_e = *reinterpret_cast<const uint16_t *>(p.exponents + (static_cast<size_t>(id) * kKvHeads + (i >> 7)) * 2);
    }
    if (kQ8 && i < 2 * static_cast<int>(kKvHeads)) sm_size[i >> 1][i & 1] = 0;
    half8_t out[2];
#pragma unroll
    for (int j = 0; j < 8; ++j) {  // as rotate_chunk rotates
        const float x = static_cast<float>(key[0][j / kElems][j % kElems]);
        const float y = static_cast<float>(key[1][j / kElems][j % kElems]);
        const float co = cs[j >> 2][j & 3], si = sn[j >> 2][j & 3];
        out[0][j] = to_h(rope ? x * co + (-y) * si : x);
        out[1][j] = to_h(rope ? y * co + x * si : y);
    }
    if constexpr (!F32) {
        if (!rope) {  // as given, bit for bit
            out[0] = key[0][0];
            out[1] = key[1][0];
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
        *reinterpret_cast<half8_t *>(&sr[kQ8 ? 1 : 0][k >> 5][(k & 31) * 8]) = v[r];
        if constexpr (kQ8) *reinterpret_cast<half8_t *>(&sr[0][tt][hh * kHeadDim + c * 8 + r * 64]) = out[r];
    }
    if (p.error_word) {
        if (!ok && i == 0) atomicOr(p.error_word, 2u);
        if (!rope && p.rope_cos != nullptr && c == 0 && hh == 0 && tt >= lo && tt < hi) atomicOr(p.error_word, 4u);
    }
    if constexpr (!kQ8) {
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
                a[e] = sr[0][e][i];
                b[e] = sr[0][e + 8][i];
            }
            *reinterpret_cast<u16x8_t *>(dst) = a;
            *reinterpret_cast<u16x8_t *>(dst + 8) = b;
        } else {
            for (int e = lo; e < hi; ++e) dst[e] = sr[0][e][i];
        }
    } else {
        __syncthreads();  // the rows are in LDS, and sm_size is cleared
        auto widen = [](uint16_t x) { return q8_value(static_cast<float>(__builtin_bit_cast(_Float16, x))); };
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            // A wave's key items are of one head; 16 lanes hold the values of one
            // head.  Sizes are not negative, so their bits are in order.
            float size = 0.f;
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int j = 0; j < 8; ++j) size = q8_size(size, q8_value(static_cast<float>(w ? v[r][j] : out[r][j])));
            size = fmaxf(size, dpp_f32<0xB1>(size));
            size = fmaxf(size, dpp_f32<0x4E>(size));
            size = fmaxf(size, dpp_f32<0x124>(size));
            size = fmaxf(size, dpp_f32<0x128>(size));
            if ((i & 15) == 0) atomicMax(&sm_size[w][w ? (i >> 4) & 1 : hh], __float_as_uint(size));
        }
        __syncthreads();
        if (!ok) return;
        const int head = i >> 7;  // of key piece i and of value row i
        int e[2], grown[2];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            e[w] = q8_exponent<CODE>(__uint_as_float(sm_size[w][head]));
            const int before = static_cast<int>((old_e >> (8 * w)) & 255) - kQ8Bias;
            if (lo > 0) e[w] = max(e[w], before);
            grown[w] = lo > 0 ? e[w] - before : 0;
        }
        {
            const int token = q8_key_token(i);
            const float inv = exp2_whole(-e[0]);
            const uint16_t *src = &sr[0][token][q8_key_dim(i)];
            const u16x8_t a = *reinterpret_cast<const u16x8_t *>(src), b = *reinterpret_cast<const u16x8_t *>(src + 8);
            q8x4_t codes;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const u16x8_t &x = w < 2 ? a : b;
                const int j = (w & 1) * 4;
                codes[w] = q8_encode<CODE>(widen(x[j]) * inv, widen(x[j + 1]) * inv, widen(x[j + 2]) * inv, widen(x[j + 3]) * inv);
            }
            if (token < lo && grown[0] > 0) {
#pragma unroll
                for (int w = 0; w < 4; ++w) codes[w] = q8_requantise<CODE>(old_k[w], grown[0]);
            }
            if (token < hi && (token >= lo || grown[0] > 0)) *reinterpret_cast<q8x4_t *>(static_cast<uint8_t *>(p.key_cache) + slab) = codes;
        }
        {
            const float inv = exp2_whole(-e[1]);
            q8x4_t codes;
#pragma unroll
            for (int w = 0; w < 4; ++w)
                codes[w] = q8_encode<CODE>(widen(sr[1][w * 4][i]) * inv, widen(sr[1][w * 4 + 1][i]) * inv, widen(sr[1][w * 4 + 2][i]) * inv,
                                           widen(sr[1][w * 4 + 3][i]) * inv);
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
            *reinterpret_cast<q8x4_t *>(static_cast<uint8_t *>(p.value_cache) + slab) = codes;
        }
        if ((i & 127) == 0)
            *reinterpret_cast<uint16_t *>(p.exponents + (static_cast<size_t>(id) * kKvHeads + head) * 2) =
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
