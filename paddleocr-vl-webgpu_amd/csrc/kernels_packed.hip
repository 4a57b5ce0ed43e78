// Causal attention of packed prompts: the rows of several sequences, each over
// its own pages (which hold the call's rows by then), behind what these held.

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "attend_device.hpp"

namespace pvlc {
namespace {

constexpr int kF16 = PVLC_HIP_KV_F16;

// A workgroup takes 32 tokens of a sequence and the 8 query heads of a kv head,
// a wave two of the heads: 64 columns.
constexpr int kWideTokens = 32, kWideWaves = 4, kWideColumns = 4;

template <bool F32>
__global__ __launch_bounds__(kWideWaves * 64, 1) void packed_wide_kernel(PackedRows p) {
    typedef std::conditional_t<F32, float, uint16_t> Element;
    const uint32_t g = blockIdx.x & 1u;
    const SeqRows q = find_share<kWideTokens, 1>(p.ragged, (gridDim.x >> 1) - 1 - (blockIdx.x >> 1));
    const int t0 = q.share * kWideTokens;
    if (!q.ok || t0 >= q.count) return;  // (the append reports it)
    const int lane = threadIdx.x & 63, row = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int h0 = static_cast<int>(g) * kGroup + wave * 2;
    const int valid = q.held + q.count;

    // Columns: head ct / 2 of the wave's, tokens t0 + ct % 2 * 16 + row (the last one again past the sequence).
    half8_t qf[kWideColumns][4];
    int limit[kWideColumns];
#pragma unroll
    for (int th = 0; th < 2; ++th) {
        const int t = min(t0 + th * 16 + row, q.count - 1);
        const int64_t at = q.begin + static_cast<int64_t>(t);
        const int64_t pos = p.positions ? p.positions[at] : q.held + static_cast<int64_t>(t);
        const bool rope = p.rope_cos != nullptr && pos >= 0 && pos < static_cast<int64_t>(p.rope_rows);
        AttendQuery<F32> raw[2][2];
        const Element *src = static_cast<const Element *>(p.query) + at * p.query_stride + h0 * kHeadDim;
#pragma unroll
        for (int hp = 0; hp < 2; ++hp)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) raw[hp][kb].load(src + hp * kHeadDim, attend_dim<kF16>(kb, kg));
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            float4_t cs[2]{}, sn[2]{};
            if (rope) {
#pragma unroll
                for (int f = 0; f < 2; ++f) {
                    cs[f] = *reinterpret_cast<const float4_t *>(p.rope_cos + pos * 64 + attend_dim<kF16>(kb, kg) + f * 4);
                    sn[f] = *reinterpret_cast<const float4_t *>(p.rope_sin + pos * 64 + attend_dim<kF16>(kb, kg) + f * 4);
                }
            }
#pragma unroll
            for (int hp = 0; hp < 2; ++hp) raw[hp][kb].rotate(rope, cs, sn, &qf[hp * 2 + th][kb], &qf[hp * 2 + th][kb + 2]);
        }
#pragma unroll
        for (int hp = 0; hp < 2; ++hp) limit[hp * 2 + th] = q.held + t + 1;
    }
    AttendPages pages;
    pages.keys = reinterpret_cast<const uint8_t *>(p.key_cache);
    pages.values = reinterpret_cast<const uint8_t *>(p.value_cache);
    pages.exponents = nullptr;
    pages.table = p.ragged.tables ? p.ragged.tables + static_cast<size_t>(q.seq) * p.ragged.max_blocks : nullptr;
    pages.first = static_cast<uint32_t>(q.seq) * p.ragged.max_blocks;
    pages.num_blocks = p.ragged.num_blocks;
    pages.head = g;
    const int keys = min(q.held + t0 + kWideTokens, valid);
    pages.last_tile = (keys - 1) >> 4;
    AttendState<kWideColumns> st;
    st.clear();
    attend<kF16, F32, kWideColumns>(pages, qf, 0, (keys + kAttendStep - 1) / kAttendStep, 1, (q.held + t0 + 1) / kAttendStep, limit, valid,
                                    p.scale_log2, st);
#pragma unroll
    for (int ct = 0; ct < kWideColumns; ++ct) {
        const float inv = 1.0f / column_sum(st.l[ct]);
        const int t = t0 + (ct & 1) * 16 + row;
        if (t < q.count) {
            Element *dst = static_cast<Element *>(p.out) + ((q.begin + static_cast<int64_t>(t)) * kQueryHeads + h0 + (ct >> 1)) * kHeadDim + kg * 4;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const float4_t v = st.o[ct][c] * inv;
                if constexpr (F32) *reinterpret_cast<float4_t *>(dst + c * 16) = v;
                else *reinterpret_cast<half4_t *>(dst + c * 16) = half4_t{to_h(v[0]), to_h(v[1]), to_h(v[2]), to_h(v[3])};
            }
        }
    }
}

}  // namespace

int launch_packed_prefill(const PackedRows &rows, void *stream) {
    PackedRows p = rows;
    p.scale_log2 = kAttendLog2e / sqrtf(static_cast<float>(kHeadDim));
    const uint32_t shares = p.ragged.rows / kWideTokens + p.ragged.num_seqs;
    hipLaunchKernelGGL(p.f32 ? packed_wide_kernel<true> : packed_wide_kernel<false>, dim3(2 * shares), dim3(kWideWaves * 64), 0,
                       static_cast<hipStream_t>(stream), p);
    return static_cast<int>(hipGetLastError());
}

}  // namespace pvlc
