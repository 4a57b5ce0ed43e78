// Moves between compact fp16 rows [tokens][2][128] and the 8-bit cache
// (pvlc_q8.hpp), through a block table.

#include <hip/hip_runtime.h>

#include <cstdint>

#include "pvlc_q8.hpp"

namespace pvlc {
namespace {

// Both kernels: a workgroup per 16-token block, both heads, through LDS, so that
// rows (512 bytes a token) and slabs (2 KiB a head) move in 16-byte pieces.
// Rows need the alignment of their elements only.  Memory bounds both: 65536
// tokens (101 MB each way) are packed in 17.3 us, 5.8 TB/s, and unpacked in 15.8 (what
// was written last is still in the Infinity Cache); 1157 tokens take 3.4 and 2.8, a
// launch and three rounds.
constexpr int kThreads = 256;
constexpr int kPad = 8;  // elements behind each LDS row of 256 dims, against bank conflicts
typedef uint16_t u16x8_any __attribute__((ext_vector_type(8), aligned(2)));

__device__ inline float widen(uint16_t x) { return q8_value(static_cast<float>(__builtin_bit_cast(_Float16, x))); }

// Key piece i (16 bytes) of a block's two slabs is head i / 128, token quad
// (i / 32) % 4, chunk (i / 4) % 8, token i % 4 of the quad; value piece i is
// (head, dim) i, all tokens.
__device__ inline int key_token(int i) { return ((i >> 5) & 3) * 4 + (i & 3); }
__device__ inline int key_dim(int i) { return (i >> 7) * kHeadDim + ((i >> 2) & 7) * 16; }

// Tokens first .. first + tokens - 1.  The block that holds `first` may hold rows
// before it (its exponents may grow with the new ones, and then those rows are
// rounded again); the codes behind the last token stay as they are.
template <int CODE>
__global__ __launch_bounds__(kThreads) void kv_pack_q8_kernel(const uint16_t *__restrict__ key_rows, const uint16_t *__restrict__ value_rows,
                                                              uint32_t first, uint32_t tokens, const int32_t *__restrict__ table,
                                                              uint32_t num_blocks, uint8_t *__restrict__ key_cache,
                                                              uint8_t *__restrict__ value_cache, uint8_t *__restrict__ exponents) {
    __shared__ __align__(16) uint16_t sr[2][kBlockTokens][kRowElems + kPad];
    __shared__ uint32_t sm_size[2][kKvHeads];
    const int i = threadIdx.x;
    const uint32_t tile = first / kBlockTokens + blockIdx.x;
    const int32_t id = table ? table[tile] : static_cast<int32_t>(tile);
    if (id < 0 || static_cast<uint32_t>(id) >= num_blocks) return;  // uniform
    // Tokens [lo, hi) of the block are new; row r of the call is token first + r.
    const int64_t base = static_cast<int64_t>(tile) * kBlockTokens - first;
    const int lo = base < 0 ? static_cast<int>(-base) : 0;
    const int hi = static_cast<int>(min(static_cast<int64_t>(kBlockTokens), static_cast<int64_t>(tokens) - base));
    if (i < 2 * static_cast<int>(kKvHeads)) sm_size[i >> 1][i & 1] = 0;
    u16x8_t piece[2][2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int k = i + r * kThreads, t = min(max(k >> 5, lo), hi - 1);  // (tokens that are not new repeat one that is)
        const size_t src = static_cast<size_t>(base + t) * kRowElems + (k & 31) * 8;
        piece[0][r] = *reinterpret_cast<const u16x8_any *>(key_rows + src);
        piece[1][r] = *reinterpret_cast<const u16x8_any *>(value_rows + src);
    }
    const size_t slab = static_cast<size_t>(id) * kKvHeads * kQ8SlabBytes + static_cast<size_t>(i) * 16;
    q8x4_t old_k{}, old_v{};
    uint32_t old_e = 0;
    const bool whole = lo == 0 && hi == static_cast<int>(kBlockTokens);  // uniform
    if (!whole) {
        old_k = *reinterpret_cast<const q8x4_t *>(key_cache + slab);
        old_v = *reinterpret_cast<const q8x4_t *>(value_cache + slab);
        old_e = *reinterpret_cast<const uint16_t *>(exponents + (static_cast<size_t>(id) * kKvHeads + (i >> 7)) * 2);
    }
    __syncthreads();  // sm_size is cleared
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        float size = 0.f;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int k = i + r * kThreads;
            *reinterpret_cast<u16x8_t *>(&sr[p][k >> 5][(k & 31) * 8]) = piece[p][r];
#pragma unroll
            for (int j = 0; j < 8; ++j) size = q8_size(size, widen(piece[p][r][j]));
        }
        // 16 lanes hold one head of a token: their largest, then one LDS atomic
        // each (sizes are not negative, so their bits are in order).
        size = fmaxf(size, dpp_f32<0xB1>(size));
        size = fmaxf(size, dpp_f32<0x4E>(size));
        size = fmaxf(size, dpp_f32<0x124>(size));
        size = fmaxf(size, dpp_f32<0x128>(size));
        if ((i & 15) == 0) atomicMax(&sm_size[p][(i >> 4) & 1], __float_as_uint(size));
    }
    __syncthreads();
    const int head = i >> 7;  // of key piece i and of value row i
    int e[2], grown[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        e[p] = q8_exponent<CODE>(__uint_as_float(sm_size[p][head]));
        const int before = static_cast<int>((old_e >> (8 * p)) & 255) - kQ8Bias;
        if (lo > 0) e[p] = max(e[p], before);
        grown[p] = lo > 0 ? e[p] - before : 0;
    }
    {
        const int t = key_token(i);
        const float inv = exp2_whole(-e[0]);
        const u16x8_t a = *reinterpret_cast<const u16x8_t *>(&sr[0][t][key_dim(i)]), b = *reinterpret_cast<const u16x8_t *>(&sr[0][t][key_dim(i) + 8]);
        q8x4_t out;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const u16x8_t &x = w < 2 ? a : b;
            const int j = (w & 1) * 4;
            out[w] = q8_encode<CODE>(widen(x[j]) * inv, widen(x[j + 1]) * inv, widen(x[j + 2]) * inv, widen(x[j + 3]) * inv);
        }
        if (t < lo && grown[0] > 0) {
#pragma unroll
            for (int w = 0; w < 4; ++w) out[w] = q8_requantise<CODE>(old_k[w], grown[0]);
        }
        if (t < hi && (t >= lo || grown[0] > 0)) *reinterpret_cast<q8x4_t *>(key_cache + slab) = out;
    }
    {
        const float inv = exp2_whole(-e[1]);
        q8x4_t out;
#pragma unroll
        for (int w = 0; w < 4; ++w)
            out[w] = q8_encode<CODE>(widen(sr[1][w * 4][i]) * inv, widen(sr[1][w * 4 + 1][i]) * inv, widen(sr[1][w * 4 + 2][i]) * inv,
                                     widen(sr[1][w * 4 + 3][i]) * inv);
        if (!whole) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const uint32_t again = grown[1] > 0 ? q8_requantise<CODE>(old_v[w], grown[1]) : old_v[w];
                uint32_t v = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int t = w * 4 + j;
                    v |= (t < lo ? again : (t < hi ? out[w] : old_v[w])) & (0xFFu << (8 * j));
                }
                out[w] = v;
            }
        }
        *reinterpret_cast<q8x4_t *>(value_cache + slab) = out;
    }
    if ((i & 127) == 0)
        *reinterpret_cast<uint16_t *>(exponents + (static_cast<size_t>(id) * kKvHeads + head) * 2) =
            static_cast<uint16_t>((e[0] + kQ8Bias) | (e[1] + kQ8Bias) << 8);
}

// Rows as fp16: code times the block's power, rounded to the nearest fp16 value
// (always one exactly, but for sizes past fp16's largest, which become it).
template <int CODE>
__global__ __launch_bounds__(kThreads) void kv_unpack_q8_kernel(const uint8_t *__restrict__ key_cache, const uint8_t *__restrict__ value_cache,
                                                                const uint8_t *__restrict__ exponents, uint32_t tokens,
                                                                const int32_t *__restrict__ table, uint32_t num_blocks,
                                                                uint16_t *__restrict__ key_rows, uint16_t *__restrict__ value_rows) {
    __shared__ __align__(16) uint16_t sr[2][kBlockTokens][kRowElems + kPad];
    const int i = threadIdx.x;
    const uint32_t t0 = blockIdx.x * kBlockTokens, ntok = min(tokens - t0, kBlockTokens);
    const int32_t id = table ? table[blockIdx.x] : static_cast<int32_t>(blockIdx.x);
    const bool ok = id >= 0 && static_cast<uint32_t>(id) < num_blocks;  // uniform; rows of a bad block are 0
    q8x4_t k{}, v{};
    uint32_t ex = kQ8Bias * 257u;
    if (ok) {
        const size_t slab = static_cast<size_t>(id) * kKvHeads * kQ8SlabBytes + static_cast<size_t>(i) * 16;
        k = *reinterpret_cast<const q8x4_t *>(key_cache + slab);
        v = *reinterpret_cast<const q8x4_t *>(value_cache + slab);
        ex = *reinterpret_cast<const uint16_t *>(exponents + (static_cast<size_t>(id) * kKvHeads + (i >> 7)) * 2);
    }
    auto half_bits = [](float x) {
        const float m = 65504.f;
        return __builtin_bit_cast(uint16_t, to_h(x != x ? x : __builtin_amdgcn_fmed3f(x, -m, m)));
    };
    const float pk = exp2_whole(static_cast<int>(ex & 255) - kQ8Bias), pv = exp2_whole(static_cast<int>(ex >> 8) - kQ8Bias);
    u16x8_t a, b;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float4_t x = q8_decode<CODE>(k[w]) * pk, y = q8_decode<CODE>(v[w]) * pv;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            (w < 2 ? a : b)[(w & 1) * 4 + j] = half_bits(x[j]);
            sr[1][w * 4 + j][i] = half_bits(y[j]);
        }
    }
    *reinterpret_cast<u16x8_t *>(&sr[0][key_token(i)][key_dim(i)]) = a;
    *reinterpret_cast<u16x8_t *>(&sr[0][key_token(i)][key_dim(i) + 8]) = b;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int piece = i + r * kThreads, t = piece >> 5;
        if (static_cast<uint32_t>(t) >= ntok) continue;
        const size_t dst = static_cast<size_t>(t0 + t) * kRowElems + (piece & 31) * 8;
        *reinterpret_cast<u16x8_any *>(key_rows + dst) = *reinterpret_cast<const u16x8_t *>(&sr[0][t][(piece & 31) * 8]);
        *reinterpret_cast<u16x8_any *>(value_rows + dst) = *reinterpret_cast<const u16x8_t *>(&sr[1][t][(piece & 31) * 8]);
    }
}

}  // namespace

int launch_kv_pack_q8(const uint16_t *key_rows, const uint16_t *value_rows, uint32_t first_token, uint32_t tokens,
                      const int32_t *table, uint32_t num_blocks, uint32_t code, uint8_t *key_cache, uint8_t *value_cache,
                      uint8_t *exponents, void *stream) {
    const uint64_t end = static_cast<uint64_t>(first_token) + tokens;
    const dim3 grid(static_cast<uint32_t>((end + kBlockTokens - 1) / kBlockTokens - first_token / kBlockTokens));
    auto *kernel = code == PVLC_HIP_KV_E4M3 ? kv_pack_q8_kernel<PVLC_HIP_KV_E4M3> : kv_pack_q8_kernel<PVLC_HIP_KV_INT8>;
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, static_cast<hipStream_t>(stream), key_rows, value_rows, first_token, tokens, table,
                       num_blocks, key_cache, value_cache, exponents);
    return static_cast<int>(hipGetLastError());
}

int launch_kv_unpack_q8(const uint8_t *key_cache, const uint8_t *value_cache, const uint8_t *exponents, uint32_t tokens,
                        const int32_t *table, uint32_t num_blocks, uint32_t code, uint16_t *key_rows, uint16_t *value_rows,
                        void *stream) {
    const dim3 grid(tokens / kBlockTokens + (tokens % kBlockTokens != 0));
    auto *kernel = code == PVLC_HIP_KV_E4M3 ? kv_unpack_q8_kernel<PVLC_HIP_KV_E4M3> : kv_unpack_q8_kernel<PVLC_HIP_KV_INT8>;
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, static_cast<hipStream_t>(stream), key_cache, value_cache, exponents, tokens, table,
                       num_blocks, key_rows, value_rows);
    return static_cast<int>(hipGetLastError());
}

}  // namespace pvlc
