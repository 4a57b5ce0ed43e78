// Rows of several sequences in one call: which sequence a workgroup's share
// belongs to, and where its rows lie in the pages.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "pvlc_device.hpp"
#include "pvlc_internal.hpp"

namespace pvlc {

struct SeqRows {
    int seq, begin, count, held;
    bool ok;    // the offsets ascend within the call's rows, and the rows fit the sequence's pages
    bool told;  // offsets of the call that the wave has seen do not: to be reported
    int share;  // the workgroup's number within the sequence
};

// Sequence of share `u` where sequence s begins at share offsets[s] / UNIT +
// SPARE * s: a closed form that leaves a sequence of n rows at least n / UNIT +
// SPARE - 1 shares, so that no workgroup has to add up the lengths before it.
// Every wave looks 64 sequences at once: one round of loads up to 64 sequences, two
// up to 4096.  Whatever the offsets hold, the sequence is one of the call's, and the
// share's number is not negative (shares before the first sequence's have no
// rows).  Of offsets that descend or leave the rows some wave is told: a window of
// the search that no wave looks into starts behind one that passes it.
// Without offsets every sequence has shares_of_each.
template <int UNIT, int SPARE>
__device__ inline SeqRows find_share(const RaggedRows &r, uint32_t u) {
    SeqRows q;
    if (!r.offsets) {
        const uint32_t per = shares_of_each<UNIT, SPARE>(r.each), s = min(u / per, r.num_seqs - 1);
        q.seq = static_cast<int>(s);
        q.begin = static_cast<int>(s * r.each);
        q.count = static_cast<int>(r.each);
        q.held = r.lens ? r.lens[s] : 0;
        q.share = static_cast<int>(u - s * per);
        q.told = false;
        q.ok = q.held >= 0 && static_cast<int64_t>(q.held) + q.count <= static_cast<int64_t>(r.max_tokens);
        return q;
    }
    const uint32_t lane = threadIdx.x & 63u;
    auto offset = [&](uint32_t s) { return r.offsets[s]; };
    auto first = [&](int32_t at, uint32_t s) { return static_cast<uint32_t>(max(at, 0)) / UNIT + SPARE * s; };
    auto inside = [&](int32_t at) { return at >= 0 && static_cast<uint32_t>(at) <= r.rows; };
    uint32_t lo = 0, n = r.num_seqs;
    q.told = false;
    while (n > 64) {
        const uint32_t stride = (n + 63) / 64, at = lane * stride;
        const int32_t start = offset(lo + min(at, n - 1));
        const uint64_t before = __ballot(at < n && first(start, lo + at) <= u);
        q.told |= __any(!inside(start) || __shfl_down(start, 1) < start) != 0;  // (the last lane meets itself)
        const uint32_t k = before ? 63 - __builtin_clzll(before) : 0;
        lo += k * stride;
        n = min(stride, n - k * stride);
    }
    const uint32_t s = lo + min(lane, n - 1);
    const int32_t a = offset(s), b = offset(s + 1), held = r.lens ? r.lens[s] : 0;
    const uint64_t before = __ballot(lane < n && first(a, s) <= u);
    const int k = before ? 63 - __builtin_clzll(before) : 0;
    q.seq = static_cast<int>(lo) + k;
    q.begin = __builtin_amdgcn_readlane(a, k);
    const int end = __builtin_amdgcn_readlane(b, k);
    q.held = __builtin_amdgcn_readlane(held, k);
    q.ok = q.begin >= 0 && end >= q.begin && static_cast<uint32_t>(end) <= r.rows && q.held >= 0;
    q.count = q.ok ? end - q.begin : 0;
    q.ok = q.ok && static_cast<int64_t>(q.held) + q.count <= static_cast<int64_t>(r.max_tokens);
    q.told |= __any(!inside(a) || !inside(b) || b < a) != 0;
    if (!before) q.count = 0;
    q.share = before ? static_cast<int>(u - first(q.begin, static_cast<uint32_t>(q.seq))) : 0;
    return q;
}

// The first workgroup of a sequence in an append (find_share<16, 2>).
__device__ inline uint32_t first_append_share(const RaggedRows &r, int seq, int begin) {
    constexpr int kTokens = kBlockTokens;
    return r.offsets ? static_cast<uint32_t>(begin) / kTokens + 2 * seq : static_cast<uint32_t>(seq) * shares_of_each<kTokens, 2>(r.each);
}

// A block of a sequence as its table gives it; outside the planes: block 0 and
// *ok false.
__device__ inline uint32_t checked_block(const RaggedRows &r, int64_t id, bool *ok) {
    *ok = id >= 0 && id < static_cast<int64_t>(r.num_blocks);
    return *ok ? static_cast<uint32_t>(id) : 0u;
}

}  // namespace pvlc
