// Packed prompts cut into items of about equal time: which workgroup takes which
// tokens and keys.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "ragged_device.hpp"

namespace pvlc {

__device__ inline PackedItem load_item(const PackedItem *items, uint32_t i) {
    PackedItem q;
    const int32_t *src = reinterpret_cast<const int32_t *>(items + i);
    q.begin = load_const(src, 0);
    q.count = load_const(src, 1);
    q.held = load_const(src, 2);
    q.seq = load_const(src, 3);
    q.t0 = load_const(src, 4);
    q.first = load_const(src, 5);
    q.end = load_const(src, 6);
    q.slot = load_const(src, 7);
    q.slots = load_const(src, 8);
    q.parts = load_const(src, 9);
    return q;
}

// A share of kPackedTokens as a whole item.
__device__ inline PackedItem packed_item(const SeqRows &s) {
    const int t0 = s.share * kPackedTokens, keys = min(s.held + t0 + kPackedTokens, s.held + s.count);
    return {s.begin, s.count, s.held, s.seq, t0, 0, (keys + 31) / 32, -1, 0, 1};
}

// By one workgroup of 256 threads.  An item longer than `most` pieces is cut
// into even parts; items are listed from the longest to the shortest (by 64
// lengths), so that workgroups, which start in this order, end together.  Which
// of equally long ones comes first, and which slots parts get, is left to
// atomics: it decides where results lie, not what they are.
__device__ inline void make_packed_plan(const RaggedRows &r, const PackedPlan &plan) {
    constexpr int kThreads = 256, kLengths = 64;
    __shared__ int32_t sm_offset[kPackedPlanSeqs + 1], sm_held[kPackedPlanSeqs];
    __shared__ uint32_t sm_length[kLengths];
    __shared__ uint32_t sm_parts;
    __shared__ unsigned long long sm_pieces;
    const int i = threadIdx.x;
    for (uint32_t s = i; s <= r.num_seqs; s += kThreads) {
        sm_offset[s] = r.offsets ? r.offsets[s] : static_cast<int32_t>(s * r.each);
        if (s < r.num_seqs) sm_held[s] = r.lens ? r.lens[s] : 0;
    }
    if (i < kLengths) sm_length[i] = 0;
    if (i == 0) {
        sm_pieces = 0;
        sm_parts = 0;
    }
    __syncthreads();
    auto first_share = [&](uint32_t s) { return static_cast<uint32_t>(max(sm_offset[s], 0)) / kPackedTokens + s; };
    const uint32_t shares = r.rows / kPackedTokens + r.num_seqs;
    auto rows_of = [&](uint32_t s) {
        SeqRows q;
        q.seq = static_cast<int>(s);
        q.begin = sm_offset[s];
        const int end = sm_offset[s + 1];
        q.held = sm_held[s];
        q.ok = q.begin >= 0 && end >= q.begin && static_cast<uint32_t>(end) <= r.rows && q.held >= 0;
        q.count = q.ok ? end - q.begin : 0;
        q.ok = q.ok && static_cast<int64_t>(q.held) + q.count <= static_cast<int64_t>(r.max_tokens);
        return q;
    };
    // The whole item of share u, if there is one.
    auto item = [&](uint32_t u, PackedItem *q) {
        uint32_t lo = 0, n = r.num_seqs;
        while (n > 1) {
            const uint32_t half = n / 2;
            if (first_share(lo + half) <= u) {
                lo += half;
                n -= half;
            } else {
                n = half;
            }
        }
        SeqRows s = rows_of(lo);
        s.share = static_cast<int>(u - first_share(lo));
        if (!s.ok || s.share < 0 || s.share >= (s.count + kPackedTokens - 1) / kPackedTokens) return false;
        *q = packed_item(s);
        return true;
    };
    PackedItem q;
    // Pieces of all items, at most: (held + 16 (k + 1) + 31) / 32 for the k-th of a sequence.
    for (uint32_t s = i; s < r.num_seqs; s += kThreads) {
        const SeqRows w = rows_of(s);
        const unsigned long long n = (w.count + kPackedTokens - 1) / kPackedTokens;
        if (w.ok && n) atomicAdd(&sm_pieces, (n * (w.held + 47ull) + 8 * n * (n - 1)) / 32 + 1);
    }
    __syncthreads();
    // A share of the pieces, in whole steps of two.  An item of
    // n > most pieces is cut into at most n / most + 1 <= 2 n / most parts, so all
    // of them into at most 2 pieces / most <= kPackedMaxParts.
    const unsigned long long share = (sm_pieces / (kPackedMaxParts / 2) + 3) / 2 * 2;
    const int most = !plan.max_parts || share > (1u << 27) ? 1 << 27 : max(static_cast<int>(share), static_cast<int>(kPackedLeastPart));
    auto parts_of = [&](const PackedItem &w) { return (w.end + most - 1) / most; };
    auto part_length = [&](const PackedItem &w, int parts) { return ((w.end + parts - 1) / parts + 1) / 2 * 2; };
    auto length_of = [&](int n) { return kLengths - 1 - min(kLengths - 1, static_cast<int>(static_cast<int64_t>(n) * kLengths / (most + 1))); };
    for (int pass = 0; pass < 2; ++pass) {
        for (uint32_t u = i; u < shares; u += kThreads) {
            if (!item(u, &q)) continue;
            const int parts = parts_of(q), each = part_length(q, parts), end = q.end;
            const int used = (end + each - 1) / each;
            if (pass == 0) {
                for (int k = 0; k < used; ++k) atomicAdd(&sm_length[length_of(min(each, end - k * each))], 1u);
                continue;
            }
            int slot = -1;
            if (used > 1) slot = static_cast<int>(atomicAdd(&sm_parts, static_cast<uint32_t>(used)));
            q.slots = max(slot, 0);
            q.parts = used;
            for (int k = 0; k < used; ++k) {
                q.first = k * each;
                q.end = min(q.first + each, end);
                q.slot = used > 1 ? slot + k : -1;
                const uint32_t at = atomicAdd(&sm_length[length_of(q.end - q.first)], 1u);
                if (at < plan.max_items) plan.items[at] = q;
            }
        }
        __syncthreads();
        if (pass == 0) {
            if (i == 0) {
                uint32_t sum = 0;
                for (int k = 0; k < kLengths; ++k) {
                    const uint32_t n = sm_length[k];
                    sm_length[k] = sum;
                    sum += n;
                }
                *plan.count = static_cast<int32_t>(min(sum, plan.max_items));
            }
            __syncthreads();
        }
    }
    for (uint32_t s = i; s < 2 * plan.max_parts; s += kThreads) plan.arrived[s] = 0;
}

}  // namespace pvlc
