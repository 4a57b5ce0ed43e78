// Device parts of the paged decode that do not depend on how the cache is
// stored: the launch's parameters, block ids, the numbering of ragged batches
// and the merge of their partitions.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "pvlc_device.hpp"
#include "pvlc_internal.hpp"

namespace pvlc {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct DecodeParams {
    uint32_t num_blocks;
    uint32_t max_blocks_per_seq;
    const int32_t *block_tables;
    const int32_t *cache_lens;
    uint32_t uniform_cache_len;
    uint16_t *key_cache;
    uint16_t *value_cache;
    const uint16_t *query;
    const uint16_t *new_key;
    const uint16_t *new_value;
    uint16_t *out;
    const float *rope_cos;
    const float *rope_sin;
    uint32_t rope_rows;
    const int32_t *positions;
    uint32_t rotate_query;
    uint32_t partition_tokens;
    uint32_t max_parts;
    uint32_t part_stride;  // partial slots per (seq, kv head): max_parts rounded up to odd
    float *part_o;      // [seq][kv head][part_stride][8 heads][128]
    float *part_ml;     // [seq][kv head][part_stride][8 heads][2]: max (log2 units), sum
    uint32_t *counters; // [seq][kv head]
    uint32_t *error_word;
    uint32_t *partition_word;  // streaming or ragged, automatic partition: receives the one used (else null)
    uint32_t compute_units;    // streaming: compute units of the device
    float scale_log2;   // log2(e)/sqrt(128)
    // f32 operands (pvlc_hip_paged_decode_f32io): query, new key and value,
    // output; null for the fp16 entry points.
    const float *query32;
    const float *new_key32;
    const float *new_value32;
    float *out32;
};

// Block ids of every tile this wave loads in one partition, one per lane:
// lane c*TILES + i holds the block of tile i of the wave's chunk c.  Tiles
// past the partition take the partition's last tile (loaded and masked).
// An id outside the planes reads block 0 and sets *bad.  One vector load
// per wave and partition, so it can be issued ahead of the key/value loads
// (or a whole work item ahead).
template <int WAVES, int TILES>
__device__ inline uint32_t wave_tile_ids(const DecodeParams &p, uint32_t s, int part_start, int part_end, int wave,
                                         bool *bad) {
    const int lane = threadIdx.x & 63;
    const int tile = (part_start >> 4) + (lane / TILES) * (WAVES * TILES) + wave * TILES + lane % TILES;
    const int t = min(tile, (part_end - 1) >> 4);
    if (p.block_tables == nullptr) return s * p.max_blocks_per_seq + static_cast<uint32_t>(t);
    const int32_t b = p.block_tables[static_cast<size_t>(s) * p.max_blocks_per_seq + t];
    const bool out = b < 0 || static_cast<uint32_t>(b) >= p.num_blocks;
    *bad = *bad || out;
    return out ? 0u : static_cast<uint32_t>(b);
}
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
constexpr int kSc1 = 16;  // cache-policy operand of the buffer intrinsics: sc1 (agent scope)

// The hand-off of a partition's partial to the workgroup that merges: without L2
// maintenance.  Partials, the arrival counter and the merge reads are relaxed
// agent-scope accesses (sc1), which are coherent across the XCDs' L2s by
// themselves; every store of the workgroup completes before its arrival is
// counted.  (A C++ release/acquire fence at agent scope would instead write back
// and invalidate the whole L2 of the XCD in every workgroup.)
//
// 8 bytes: two floats, as atomics.  16 bytes: elements of a unit's partials (a
// sequence's kv head), through the compiler's buffer intrinsics so that its waits
// cover them.
__device__ inline void store_pair_sc1(float *q, float lo, float hi) {
    __hip_atomic_store(reinterpret_cast<uint64_t *>(q),
                       static_cast<uint64_t>(__float_as_uint(lo)) | (static_cast<uint64_t>(__float_as_uint(hi)) << 32),
                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline void load_pair_sc1(const float *q, float *lo, float *hi) {
    const uint64_t v =
        __hip_atomic_load(reinterpret_cast<const uint64_t *>(q), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *lo = __uint_as_float(static_cast<uint32_t>(v));
    *hi = __uint_as_float(static_cast<uint32_t>(v >> 32));
}
// Raw buffer over the unit's partials: stride 0, 2^31 - 1 bytes, and the fourth
// descriptor word of a raw 32-bit-element buffer on gfx9-family parts (data
// format 32 in bits 15-18).
__device__ inline __amdgpu_buffer_rsrc_t partials_buffer(const DecodeParams &p, size_t unit) {
    return __builtin_amdgcn_make_buffer_rsrc(p.part_o + unit * (kGroup * kHeadDim), 0, 0x7fffffff, 0x00020000);
}
__device__ inline void store_partial_sc1(__amdgpu_buffer_rsrc_t rsrc, uint32_t element, u32x4_t v) {
    __builtin_amdgcn_raw_buffer_store_b128(v, rsrc, static_cast<int>(element * 4), 0, kSc1);
}
__device__ inline u32x4_t load_partial_sc1(__amdgpu_buffer_rsrc_t rsrc, uint32_t element) {
    return __builtin_amdgcn_raw_buffer_load_b128(rsrc, static_cast<int>(element * 4), 0, kSc1);
}
// Counts the workgroup's partition as arrived; whether it is the last of its
// unit, the same for every thread (sm_last is LDS).  Every thread calls it.
__device__ inline bool last_to_arrive(const DecodeParams &p, uint32_t s, uint32_t g, uint32_t part, int num_parts, int &sm_last) {
    // Wait for this wave's partial stores to complete (a single-wave
    // workgroup's __syncthreads() emits no wait), then for every wave.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    // Arrival, counted in generations (kArrivalSpan): the partition with the
    // highest index adds kArrivalSpan - (num_parts - 1), the others 1, so the
    // arrival that completes a multiple of kArrivalSpan is the last one, and
    // the counter is left ready for the next launch without a reset.
    if (threadIdx.x == 0) {
        const uint32_t inc =
            part == static_cast<uint32_t>(num_parts - 1) ? kArrivalSpan - static_cast<uint32_t>(num_parts - 1) : 1u;
        const uint32_t prev =
            __hip_atomic_fetch_add(p.counters + s * kKvHeads + g, inc, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        sm_last = ((prev + inc) & (kArrivalSpan - 1)) == 0;
    }
    __syncthreads();
    return sm_last;
}
// Cache length of sequence s if it is valid for this launch (one row to
// append, inside the block table and the partitions of the workspace), else -1.
__device__ inline int64_t checked_cache_len(const DecodeParams &p, int64_t len) {
    const int64_t capacity = static_cast<int64_t>(p.max_blocks_per_seq) * 16;
    const int64_t span = static_cast<int64_t>(p.max_parts) * p.partition_tokens;
    return (len < 0 || len + 1 > capacity || len + 1 > span) ? -1 : len;
}

// x / d for integers 0 <= x, x + d < 2^19, 1 <= d <= 4096, x / d <= 2^19 / d:
// the reciprocal (1 ulp) and the product move (x + 0.5) / d by less than
// 2^19 / d 2^-22 < 0.25 / d, and it lies 0.5 / d or more from an integer.
// Five instructions where a 32-bit division takes about thirty.
__device__ inline uint32_t small_quotient(uint32_t x, uint32_t d) {
    return static_cast<uint32_t>((static_cast<float>(x) + 0.5f) * __builtin_amdgcn_rcpf(static_cast<float>(d)));
}

// Partitions of P tokens that the len + 1 rows of a sequence take (at most
// kMaxMergeParts of 4096: checked_cache_len).
__device__ inline uint32_t partitions_of(int64_t len, uint32_t P) {
    return small_quotient(static_cast<uint32_t>(len) + P, P);
}

// Inclusive prefix sum over the lanes of a wave.
__device__ inline uint32_t wave_inclusive_scan(uint32_t x) {
#define PVLC_SCAN_STEP(CTRL, ROWS) x += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, ROWS, 0xf, false))
    PVLC_SCAN_STEP(0x111, 0xf);  // row_shr 1, 2, 4, 8 within each 16 lanes
    PVLC_SCAN_STEP(0x112, 0xf);
    PVLC_SCAN_STEP(0x114, 0xf);
    PVLC_SCAN_STEP(0x118, 0xf);
    PVLC_SCAN_STEP(0x142, 0xa);  // lane 15 of rows 0 and 2 to rows 1 and 3
    PVLC_SCAN_STEP(0x143, 0xc);  // lane 31 to rows 2 and 3
#undef PVLC_SCAN_STEP
    return x;
}
// Exclusive scan of one int per thread over the workgroup; *total receives
// the sum.
template <int kThreads>
__device__ inline int workgroup_exclusive_scan(int v, int *sm_wave_sums, int *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    if (lane == 63) sm_wave_sums[wave] = x;
    __syncthreads();
    int before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) {
        const int t = sm_wave_sums[w];
        before += w < wave ? t : 0;
        sum += t;
    }
    __syncthreads();
    *total = sum;
    return before + x - v;
}
// Persistent grid for ragged lengths and long contexts: every workgroup
// reads the cache lengths (and positions) once, into registers or LDS, numbers the
// (sequence, partition, kv head) items that hold rows, and walks items blockIdx.x,
// blockIdx.x + gridDim.x, ...  Sequences with fewer partitions launch no
// empty workgroups, so every compute unit stays on real work, and the block
// ids of the next item are loaded while the current one runs.
// TILES: 16-token tiles a wave holds at once; run_item(P, s, g, part, len, pos,
// ids, ids_bad) runs one item.
template <int WAVES, int TILES, class RunItem>
__device__ inline void ragged_items(const DecodeParams &p, uint32_t num_seqs, RunItem run_item) {
    constexpr int kThreads = WAVES * 64;
    __shared__ int sm_first[kMaxRaggedSeqs + 1];  // first item (per kv head) of each sequence
    __shared__ int sm_len[kMaxRaggedSeqs];        // cache length, -1 if invalid
    __shared__ int sm_pos[kMaxRaggedSeqs];        // rotary position of the appended row
    __shared__ int sm_wave_sums[WAVES];
    __shared__ uint32_t sm_counts[kPartitionChoices][WAVES];
    const int n = static_cast<int>(num_seqs);
    // Validity is judged against the partition the host planned with.
    const int P0 = static_cast<int>(p.partition_tokens);
    static_assert(TILES == 2 || TILES == 4, "the block ids of 64 tiles a wave cover streaming_span");
    constexpr uint32_t kSpan = streaming_span(WAVES);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const uint32_t units = max(1u, p.compute_units);
    // Automatic partition (choose_streaming_partition): item k runs on
    // workgroup k mod grid, and the grid fills every compute unit before it
    // doubles up, so item k lands on unit k mod units and a unit streams
    // ceil(items / units) items one after the other at the per-unit HBM rate.
    // Every workgroup computes the same counts from the same lengths.  The
    // candidates stop at kSpan, the tokens covered by the block ids the
    // workgroup's waves hold (wave_tile_ids).
    auto choose = [&](const uint32_t (&counts)[kPartitionChoices]) {  // partitions at each candidate
        uint32_t turns[kPartitionChoices];
#pragma unroll
        for (int c = 0; c < kPartitionChoices; ++c) {
            // at most 2048 sequences x 64 partitions x 2 heads, 4096 units
            turns[c] = __builtin_amdgcn_readfirstlane(small_quotient(counts[c] * kKvHeads + units - 1, units));
        }
        const uint32_t best = best_streaming_partition(turns, static_cast<uint32_t>(P0), kSpan);
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            p.partition_word[0] = best;
            p.partition_word[1] = units;  // for inspection
        }
        return static_cast<int>(__builtin_amdgcn_readfirstlane(best));  // uniform: keep the item arithmetic scalar
    };
    // Up to a wave's lanes of sequences every wave numbers them by itself, one
    // per lane: no LDS and no barrier ahead of the first loads.  (Through LDS,
    // with 64-bit divisions for the candidates, this prologue took 2.5 us more
    // of every launch: 18 caches of 4096 rows 19.1 -> 16.6 us, 13 sequences up
    // to 4096 rows 15.0 -> 12.6.  Several sequences per lane, for launches of
    // up to 256, cost the small ones 0.8 us and won nothing.)
    const bool in_lanes = n <= 64;  // uniform
    int P = P0, total = 0;
    int lane_len = -1, lane_pos = 0, lane_first = 0;
    if (in_lanes) {
        if (lane < n) {
            lane_len = static_cast<int>(
                checked_cache_len(p, p.cache_lens ? p.cache_lens[lane] : static_cast<int64_t>(p.uniform_cache_len)));
            lane_pos = p.positions ? p.positions[lane] : lane_len;
            if (lane_len < 0 && blockIdx.x == 0 && wave == 0) atomicOr(p.error_word, 1u);
        }
        auto parts_at = [&](uint32_t pc) { return lane_len < 0 || pc == 0 ? 0u : partitions_of(lane_len, pc); };
        if (p.partition_word) {
            uint32_t counts[kPartitionChoices];
#pragma unroll
            for (int c = 0; c < kPartitionChoices; ++c) {
                const uint32_t x =
                    wave_inclusive_scan(parts_at(streaming_partition_candidate(static_cast<uint32_t>(P0), c, kSpan)));
                counts[c] = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x), 63));
            }
            P = choose(counts);
        }
        const uint32_t parts = parts_at(static_cast<uint32_t>(P)), through = wave_inclusive_scan(parts);
        lane_first = static_cast<int>(through - parts);
        total = __builtin_amdgcn_readlane(static_cast<int>(through), 63);
    } else {
        const int per = (n + kThreads - 1) / kThreads;
        const int i0 = static_cast<int>(threadIdx.x) * per;
        uint32_t counts[kPartitionChoices] = {};
        for (int i = i0; i < min(i0 + per, n); ++i) {
            const int64_t len =
                checked_cache_len(p, p.cache_lens ? p.cache_lens[i] : static_cast<int64_t>(p.uniform_cache_len));
            if (len < 0 && blockIdx.x == 0) atomicOr(p.error_word, 1u);
            sm_len[i] = static_cast<int>(len);
            sm_pos[i] = p.positions ? p.positions[i] : static_cast<int>(len);
            if (p.partition_word) {
#pragma unroll
                for (int c = 0; c < kPartitionChoices; ++c) {
                    const uint32_t pc = streaming_partition_candidate(static_cast<uint32_t>(P0), c, kSpan);
                    counts[c] += len < 0 || pc == 0 ? 0u : partitions_of(len, pc);
                }
            }
        }
        if (p.partition_word) {
#pragma unroll
            for (int c = 0; c < kPartitionChoices; ++c) {
                const uint32_t x = wave_inclusive_scan(counts[c]);
                if (lane == 63) sm_counts[c][wave] = x;
            }
            __syncthreads();
#pragma unroll
            for (int c = 0; c < kPartitionChoices; ++c) {
                counts[c] = 0;
#pragma unroll
                for (int w = 0; w < WAVES; ++w) counts[c] += sm_counts[c][w];
            }
            P = choose(counts);
        }
        int local = 0;
        for (int i = i0; i < min(i0 + per, n); ++i) {
            const int len = sm_len[i];  // written by this thread above
            const int parts = len < 0 ? 0 : static_cast<int>(partitions_of(len, static_cast<uint32_t>(P)));
            sm_first[i + 1] = parts;
            local += parts;
        }
        int run = workgroup_exclusive_scan<kThreads>(local, sm_wave_sums, &total);
        for (int i = i0; i < min(i0 + per, n); ++i) {
            run += sm_first[i + 1];
            sm_first[i + 1] = run;
        }
        if (threadIdx.x == 0) sm_first[0] = 0;
        __syncthreads();
    }

    // Item k (per kv head) lies in the last sequence s with first[s] <= k
    // (sequences without partitions share their successor's start).
    auto locate = [&](int k, uint32_t *s_out, uint32_t *part_out, int *len_out) {
        if (in_lanes) {
            const int s = __popcll(__ballot(lane < n && lane_first <= k)) - 1;  // the lanes 0 .. s
            *s_out = static_cast<uint32_t>(s);
            *part_out = static_cast<uint32_t>(k - __builtin_amdgcn_readlane(lane_first, s));
            *len_out = __builtin_amdgcn_readlane(lane_len, s);
            return;
        }
        int lo = 0, hi = n - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (sm_first[mid] <= k) lo = mid;
            else hi = mid - 1;
        }
        *s_out = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(lo));
        *part_out = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(k - sm_first[lo]));
        *len_out = __builtin_amdgcn_readfirstlane(sm_len[lo]);
    };
    const int items = total * static_cast<int>(kKvHeads);
    int item = blockIdx.x;
    if (item >= items) return;
    uint32_t s = 0, part = 0;
    int len = 0;
    locate(item >> 1, &s, &part, &len);
    bool bad = false;
    uint32_t ids = wave_tile_ids<WAVES, TILES>(p, s, static_cast<int>(part) * P,
                                               min(static_cast<int>(part + 1) * P, len + 1), wave, &bad);
    for (;;) {
        const int next = item + static_cast<int>(gridDim.x);
        uint32_t s_next = 0, part_next = 0, ids_next = 0;
        int len_next = 0;
        bool bad_next = false;
        if (next < items) {
            locate(next >> 1, &s_next, &part_next, &len_next);
            ids_next = wave_tile_ids<WAVES, TILES>(p, s_next, static_cast<int>(part_next) * P,
                                                   min(static_cast<int>(part_next + 1) * P, len_next + 1), wave,
                                                   &bad_next);
        }
        const int pos = in_lanes ? __builtin_amdgcn_readlane(lane_pos, static_cast<int>(s)) : sm_pos[s];
        run_item(P, s, static_cast<uint32_t>(item & 1), part, len, pos, ids, bad);
        if (next >= items) break;
        __syncthreads();  // the next item reuses the workgroup's LDS
        item = next;
        s = s_next;
        part = part_next;
        len = len_next;
        ids = ids_next;
        bad = bad_next;
    }
}
// LSE merge of the partials the ragged kernel stored: one workgroup per
// (kv head, sequence); each thread folds 4 consecutive output elements of one
// head over every partition, 16 partitions per batch of loads.  Sequences of
// one partition were written directly by the ragged kernel.
template <bool F32IO>
__global__ __launch_bounds__(256) void paged_decode_merge_kernel(DecodeParams p) {
    const uint32_t g = blockIdx.x;
    const uint32_t s = blockIdx.y;
    const int64_t len = checked_cache_len(
        p, p.cache_lens ? load_const(p.cache_lens, s) : static_cast<int64_t>(p.uniform_cache_len));
    if (len < 0) return;
    // The ragged kernel wrote the partition it used before this launch began.
    const int P = static_cast<int>(p.partition_word ? load_const(reinterpret_cast<const int32_t *>(p.partition_word), 0)
                                                    : p.partition_tokens);
    const int num_parts = static_cast<int>(partitions_of(len, static_cast<uint32_t>(P)));
    if (num_parts <= 1) return;
    const int e0 = threadIdx.x * 4;
    const int h = e0 >> 7;
    const size_t unit = (static_cast<size_t>(s) * kKvHeads + g) * p.part_stride;
    const float *all_o = p.part_o + unit * (kGroup * kHeadDim);
    const float *all_ml = p.part_ml + unit * (2 * kGroup);
    constexpr int kBatch = 16;
    float Mg = -INFINITY, Lg = 0.f;
    float4_t og = float4_t{0.f, 0.f, 0.f, 0.f};
    for (int q0 = 0; q0 < num_parts; q0 += kBatch) {
        float mv[kBatch], lv[kBatch];
        float4_t ov[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const int q = min(q0 + b, num_parts - 1);  // clamped re-reads get weight 0 below
            mv[b] = all_ml[q * (2 * kGroup) + 2 * h];
            lv[b] = all_ml[q * (2 * kGroup) + 2 * h + 1];
            ov[b] = *reinterpret_cast<const float4_t *>(all_o + static_cast<size_t>(q) * (kGroup * kHeadDim) + e0);
        }
        float Mb = Mg;
#pragma unroll
        for (int b = 0; b < kBatch; ++b)
            if (q0 + b < num_parts) Mb = fmaxf(Mb, mv[b]);  // finite: every partition holds a token
        const float a = __builtin_amdgcn_exp2f(Mg - Mb);   // 0 on the first batch
        Lg *= a;
        og *= a;
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const float w = (q0 + b < num_parts) ? __builtin_amdgcn_exp2f(mv[b] - Mb) : 0.f;
            Lg += lv[b] * w;
            og += ov[b] * w;
        }
        Mg = Mb;
    }
    const float inv = 1.0f / Lg;
    const size_t out_off = (static_cast<size_t>(s) * kQueryHeads + g * kGroup) * kHeadDim + e0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (F32IO) p.out32[out_off + e] = og[e] * inv;
        else p.out[out_off + e] = __builtin_bit_cast(uint16_t, to_h(og[e] * inv));
    }
}

}  // namespace
}  // namespace pvlc
