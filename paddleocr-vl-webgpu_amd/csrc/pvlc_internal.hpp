// Internal declarations shared by the pvlc_hip translation units.
#pragma once

#include <cstddef>
#include <cstdint>
#include <string>

#include "pvlc_hip.h"

namespace pvlc {

constexpr uint32_t kQueryHeads = PVLC_HIP_QUERY_HEADS;
constexpr uint32_t kKvHeads = PVLC_HIP_KV_HEADS;
constexpr uint32_t kHeadDim = PVLC_HIP_HEAD_DIM;
constexpr uint32_t kGroup = kQueryHeads / kKvHeads;
constexpr uint32_t kBlockTokens = PVLC_HIP_BLOCK_TOKENS;
constexpr uint32_t kRowElems = kKvHeads * kHeadDim;          // one cache row, both heads
constexpr uint32_t kBlockHeadElems = kBlockTokens * kHeadDim;  // one (block, head) slab

// Key slot of token t (0..15) inside a 16-token block of the key plane: bits
// 2 and 3 of t swapped, so that slots 0-7 hold tokens 0-3 and 8-11 and slots
// 8-15 tokens 4-7 and 12-15.  With this order one 16x16x32 score MFMA over
// rows "slots 0-7 of tile A, slots 0-7 of tile B" (and a second over slots
// 8-15) leaves each lane the scores of 8 consecutive tokens of one tile:
// exactly the probability operand of a 16x16x32 P.V MFMA whose values are
// 16-byte loads.  The map is its own inverse (constexpr: usable on host and
// device).
constexpr int key_slot(int t) { return (t & 3) | ((t & 4) << 1) | ((t & 8) >> 1); }
constexpr uint32_t kMaxDecoderHeadDim = 128;                   // runtime-core lib.rs:180
constexpr uint32_t kMaxWebgpuDispatch = 65535;                 // runtime-core lib.rs:187
constexpr uint32_t kMaxMergeParts = 64;  // split-K partitions one in-kernel merge combines
// Automatic partitioning: workgroups one launch aims to keep resident (one
// per MI355X compute unit), the most tiles one workgroup covers without
// looping (12 waves x one pair of tiles), and the most partitions of the
// balanced rule.
constexpr uint32_t kTargetWorkgroups = 256;
constexpr uint32_t kSingleShotTiles = 24;
constexpr uint32_t kMaxBalancedParts = 16;
// Arrival counters of the single-shot split-K hand-off count in generations:
// every partition adds 1 except the one with the highest index, which adds
// kArrivalSpan - (parts - 1), so a launch adds exactly kArrivalSpan to the
// counter of each (sequence, kv head) it merges.  The counter is never reset:
// the arrival that brings it to a multiple of kArrivalSpan is the last, and
// any value is ready for the next launch (a power of two above the 64
// partitions a merge combines, so the arithmetic holds modulo 2^32).
constexpr uint32_t kArrivalSpan = 1024;
static_assert((kArrivalSpan & (kArrivalSpan - 1)) == 0 && kArrivalSpan > 64, "arrival span");
// Sequences the ragged (persistent) decode kernel numbers in LDS; launches
// with more ragged sequences use one workgroup per (partition, head, sequence).
constexpr uint32_t kMaxRaggedSeqs = 2048;

// Automatic streaming partition.  The host plans p0; the streaming kernel may
// lengthen it to a candidate p0 + c*step (c < kPartitionChoices, step = p0/4
// rounded down to 16 tokens, at least 16), never beyond the span one
// workgroup of the streaming shape covers: a wave keeps the block ids of its
// tiles one per lane (64 lanes = 32 chunks of 2 tiles), and a chunk round of
// `waves` waves covers waves x 2 tiles, so a partition spans at most
// 32 x waves x 2 x 16 = 1024 x waves tokens (4096 for the 4-wave shape).
// Candidates beyond the span are skipped (0 below).
constexpr int kPartitionChoices = 5;
constexpr uint32_t streaming_span(uint32_t waves) { return 1024u * waves; }
constexpr uint32_t streaming_partition_candidate(uint32_t p0, int c, uint32_t span) {
    const uint32_t quarter = (p0 / 4) & ~15u;
    const uint32_t pc = p0 + static_cast<uint32_t>(c) * (quarter > 16 ? quarter : 16);
    return pc <= span ? pc : 0;
}
// The candidate with the least turns * P (the first on ties), where turns[c] =
// ceil(items / units) at candidate c and items counts its (sequence, partition,
// kv head) items: item k runs on compute unit k mod units, so a unit streams
// `turns` partitions one after the other.  p0 itself is a candidate whenever
// p0 <= span, which the host's shape choice guarantees.
constexpr uint32_t best_streaming_partition(const uint32_t (&turns)[kPartitionChoices], uint32_t p0, uint32_t span) {
    uint32_t best_p = p0;
    uint64_t best = ~0ull;
    for (int c = 0; c < kPartitionChoices; ++c) {
        const uint32_t pc = streaming_partition_candidate(p0, c, span);
        if (pc == 0) continue;
        const uint64_t cost = static_cast<uint64_t>(turns[c]) * pc;
        if (cost < best) {
            best = cost;
            best_p = pc;
        }
    }
    return best_p;
}
constexpr uint32_t choose_streaming_partition(const uint32_t (&items)[kPartitionChoices], uint32_t p0,
                                              uint32_t units, uint32_t span) {
    const uint32_t u = units > 0 ? units : 1;
    uint32_t turns[kPartitionChoices] = {};
    for (int c = 0; c < kPartitionChoices; ++c) turns[c] = (items[c] + u - 1) / u;
    return best_streaming_partition(turns, p0, span);
}

// Status of a failed call: RuntimeErrorCode in bits 8..15, InvocationErrorCode
// in bits 0..7; records the message for pvlc_hip_last_error_message().
pvlc_hip_status fail(int runtime_code, int invocation_code, const std::string &message);
inline pvlc_hip_status invalid(int invocation_code, const std::string &message) {
    return fail(PVLC_HIP_INVALID_INVOCATION, invocation_code, message);
}
pvlc_hip_status ok();

// Plan-layer error: an InvocationErrorCode plus message (runtime-core's
// InvocationError, lib.rs:5365-5395).
struct PlanError {
    int code = PVLC_HIP_INV_NONE;
    std::string message;
    explicit operator bool() const { return code != PVLC_HIP_INV_NONE; }
};

PlanError plan_session_geometry(uint32_t query_heads, uint32_t key_value_heads, uint32_t head_dim,
                                uint32_t prefix_tokens, uint32_t cache_capacity, pvlc_hip_kv_session_plan *out);
PlanError plan_split(uint32_t cache_tokens, uint32_t query_heads, uint32_t key_value_heads, uint32_t head_dim,
                     pvlc_hip_gqa_split_plan *out);
PlanError plan_descriptor(const pvlc_hip_kv_session_descriptor *d, pvlc_hip_kv_session_plan *out);
PlanError plan_step(const pvlc_hip_kv_session_plan *plan, uint32_t cache_tokens, const pvlc_hip_kv_step_operands *step,
                    pvlc_hip_kv_step_plan *out);
PlanError plan_cached_gqa(const pvlc_hip_cached_gqa_invocation *inv, pvlc_hip_kv_session_plan *session_out,
                          pvlc_hip_kv_step_plan *step_out);

// fp16 storage admits only values whose RNE rounding is finite (|x| < 65520).
bool fp16_representable(const float *values, size_t n);
uint16_t f32_to_f16_rne(float value);
float f16_to_f32(uint16_t bits);

// Host copies between the compact reference rows [tokens][2][128] and the
// blocked device layout (contiguous blocks 0..ceil(tokens/16)-1).
size_t key_blocked_index(uint32_t token, uint32_t head, uint32_t dim);
size_t value_blocked_index(uint32_t token, uint32_t head, uint32_t dim);
// The fp16 slabs (both heads) of one 16-token block from its compact f32 rows
// [tokens][2][128], tokens of 1..16, rounded as f32_to_f16_rne rounds (the
// other tokens are zero).
void key_block_slabs(const float *rows, uint32_t tokens, uint16_t *slabs);
void value_block_slabs(const float *rows, uint32_t tokens, uint16_t *slabs);

// Kernel launchers (kernels_*.hip).  Return hipError_t as int.
// The f32 operands of pvlc_hip_paged_decode_f32io (device pointers).
struct DecodeOperands32 {
    const float *query;      // [num_seqs][16][128]
    const float *new_key;    // [num_seqs][2][128]
    const float *new_value;  // [num_seqs][2][128]
    float *out;              // [num_seqs][16][128]
};
struct DecodeLaunch {
    const pvlc_hip_paged_decode_args *args;
    uint32_t partition_tokens;
    uint32_t waves;      // waves per workgroup
    uint32_t pairs;      // pairs of 16-token tiles a wave holds per chunk
    bool streaming;      // persistent kernel + merge kernel (else one workgroup per partition)
    uint32_t max_parts;
    uint32_t part_stride;
    float *part_o;
    float *part_ml;
    uint32_t *counters;
    uint32_t *error_word;
    // Streaming regime with an automatic partition: the persistent kernel may
    // lengthen the partition to fill its last round of items and writes the
    // partition it used here for the merge kernel, and the compute units it
    // assumed in the next word (null: partition_tokens as is).  A ragged
    // automatic launch of the single-shot kernel records its partition here too.
    uint32_t *partition_word;
    // f32 operands instead of args' fp16 query, new key and value, output
    // (null: the fp16 ones).
    const DecodeOperands32 *f32 = nullptr;
};
int launch_paged_decode(const DecodeLaunch &launch, void *stream);
// Workgroups of `kernel` the current device keeps resident at once, at most
// max_items; *units receives its compute units (kernels_decode.hip).
uint32_t resident_workgroups(const void *kernel, int threads, uint64_t max_items, uint32_t *units, int *err);

// The 8-bit cache: bytes of one (block, head) of a plane, the bias of a stored
// exponent, and the least exponent (an fp16 value's size is at least 2^-24, so
// its codes reach down to 2^-33; a block of zeros has the least).
constexpr uint32_t kQ8SlabBytes = kBlockHeadElems;
constexpr int kQ8Bias = 127;
constexpr int kQ8LeastExponent = -32;
struct DecodeCodes {
    uint32_t code;        // PVLC_HIP_KV_E4M3 or PVLC_HIP_KV_INT8
    uint8_t *exponents;   // [block][kv head][key, value]
};
// Single-shot shapes of the 8-bit decode: a wave for each 64 tokens of a
// partition, up to 768 (the fp16 cache's largest shape in bytes).
constexpr uint32_t kQ8Shapes[] = {1, 2, 3, 4, 6, 8, 12};
constexpr uint32_t kQ8SingleShotTiles = 48;
constexpr uint32_t q8_waves(uint32_t partition_tokens) {
    for (uint32_t w : kQ8Shapes)
        if (partition_tokens <= w * 64) return w;
    return kQ8Shapes[6];
}
// Whether a launch of these partitions a sequence takes the persistent kernel.
bool q8_streams(uint32_t partition_tokens, uint64_t parts, uint32_t num_seqs, bool ragged);
// Partition of an automatic 8-bit decode of `rows` tokens a sequence (an upper
// bound of them when ragged), with at most workspace_parts partitions.
uint32_t q8_auto_partition(uint32_t num_seqs, uint32_t rows, bool ragged, uint32_t workspace_parts);
int launch_paged_decode_q8(const DecodeLaunch &launch, const DecodeCodes &codes, void *stream);
int launch_kv_pack_q8(const uint16_t *key_rows, const uint16_t *value_rows, uint32_t first_token, uint32_t tokens,
                      const int32_t *table, uint32_t num_blocks, uint32_t code, uint8_t *key_cache, uint8_t *value_cache,
                      uint8_t *exponents, void *stream);
int launch_kv_unpack_q8(const uint8_t *key_cache, const uint8_t *value_cache, const uint8_t *exponents, uint32_t tokens,
                        const int32_t *table, uint32_t num_blocks, uint32_t code, uint16_t *key_rows, uint16_t *value_rows,
                        void *stream);
int launch_fill_u32(uint32_t *dst, size_t words, uint32_t value, void *stream);
int launch_kv_pack(const uint16_t *key_rows, const uint16_t *value_rows, uint32_t tokens, const int32_t *table,
                   uint32_t num_blocks, uint16_t *key_cache, uint16_t *value_cache, uint32_t *error_word,
                   void *stream);
int launch_kv_unpack(const uint16_t *key_cache, const uint16_t *value_cache, uint32_t tokens, const int32_t *table,
                     uint32_t num_blocks, uint16_t *key_rows, uint16_t *value_rows, void *stream);
// The f32 operands of pvlc_hip_paged_prefill_f32io (device pointers).
struct PrefillOperands32 {
    const float *query;  // [tokens][16][128]
    const float *key;    // [tokens][2][128]
    const float *value;  // [tokens][2][128]
    float *out;          // [tokens][16][128]
};
int launch_prefill(const pvlc_hip_paged_prefill_args *args, void *stream, const PrefillOperands32 *f32 = nullptr);

// Rows of several sequences in one call (ragged_device.hpp): those of sequence
// s are offsets[s] .. offsets[s + 1] - 1 (without offsets: `each` rows apiece),
// and its pages hold lens[s] rows before them (without lens: none).
struct RaggedRows {
    uint32_t num_seqs, rows, each;
    const int32_t *offsets, *lens;
    uint32_t num_blocks, max_blocks;
    const int32_t *tables;
    uint32_t max_tokens;  // that a sequence may come to hold
};
// Shares of UNIT rows that n rows take: with SPARE 1 from their own first row
// on, with SPARE 2 from any row of a share on.
template <int UNIT, int SPARE>
constexpr uint32_t shares_of_each(uint32_t n) {
    return SPARE == 2 ? (n + UNIT - 2) / UNIT + 1 : (n + UNIT - 1) / UNIT;
}
// Packed prompts: 16 tokens t0 .. of a sequence (its rows begin at `begin`) and
// the pieces of 32 keys that one workgroup takes; slot: where it leaves a part of
// an item (-1: it has all of them), among the slots slots .. slots + parts - 1.
constexpr int kPackedTokens = 16;
struct PackedItem {
    int32_t begin, count, held, seq, t0, first, end, slot, slots, parts;
};
// Where an append's launch leaves a plan of items (items null: it makes none).
struct PackedPlan {
    int32_t *count;
    PackedItem *items;
    uint32_t *arrived;  // [slot][kv head], cleared: parts that have been left
    uint32_t max_items, max_parts;
};
// Rows appended to their pages (kernels_append.hip); strides in elements.
struct AppendRows {
    RaggedRows ragged;
    uint32_t code;
    bool f32;
    const void *key, *value;
    int64_t key_stride, value_stride;
    const float *rope_cos, *rope_sin;
    uint32_t rope_rows;
    const int32_t *positions;
    void *key_cache, *value_cache;
    uint8_t *exponents;
    uint32_t *error_word;
    PackedPlan plan;
    uint32_t *odd;  // [workgroup] or null: not 0 where a block's values are not all finite
};
int launch_kv_append(const AppendRows &rows, void *stream);
// Packed prompts over pages that hold their rows (kernels_packed.hip).
struct PackedRows {
    RaggedRows ragged;
    bool f32;
    const void *query;
    void *out;
    int64_t query_stride;
    const float *rope_cos, *rope_sin;
    uint32_t rope_rows;
    const int32_t *positions;
    const uint16_t *key_cache, *value_cache;
    uint32_t *error_word;
    float scale_log2;
    // The plan that the append's launch made (items null: none), and what bounds
    // its items.
    const int32_t *count;
    const PackedItem *items;
    uint32_t *arrived;
    uint64_t *partials;  // [slot][kv head][kPackedPartPairs]
    const int32_t *odd;
    uint32_t max_items;
    bool narrow;  // one head a workgroup, without a plan
};
int launch_packed_prefill(const PackedRows &rows, void *stream);
// Calls of few tokens over short contexts give a workgroup one head, not eight:
// eight times the workgroups and no plan, but every head reads its keys again.
// Whole calls, us, one head against eight: a prompt of 16 tokens 7.9 against 12.4,
// of 500 tokens 12.2 against 21.1; 16 tokens each on 500 held, 16 sequences 11.9
// against 22.2, 32 sequences 18.5 against 23.1, 64 (128 shares) 27.4 against 25.1;
// on 4000 held, 4 sequences 18.9 against 30.6, 16 (32 shares) 39.4 against 37.5;
// 1000 tokens on 1000 held 34.9 against 44.8.
constexpr uint32_t kNarrowShares = 72, kNarrowContext = 4096, kNarrowRows = 128000;
inline bool packed_is_narrow(uint32_t num_seqs, uint32_t rows, uint32_t max_context) {
    const uint64_t shares = static_cast<uint64_t>(rows / kPackedTokens) + num_seqs;
    return shares <= kNarrowShares && max_context <= kNarrowContext && shares * max_context <= kNarrowRows;
}
// Its workspace: 256 bytes of words (0 the error word, 1 the plan's count), room for the
// paged decodes' arrival counters, which are never cleared (a workspace may serve
// both, and lies off them here), what the append says of its blocks, the items, the counts of
// parts that have been left, and the parts.  More sequences than kPackedPlanSeqs (what the plan holds in LDS) are not planned.  Items are cut
// from kPackedLeastPart pieces on, or from what lets the cut items of a call have
// kPackedMaxParts parts at most, 1.28 times what each of the 512 resident
// workgroups would have of an even share.  256 / 400 / 512 / 640 / 768 / 1024 parts: 12
// prompts of 211 to 2010 tokens 79 / 78 / 82 / 86 / 89 / 97 us, 6 chunks of 256 to 512
// tokens on 16384 rows 221 / 197 / 213 / 201 / 214 / 216.  (All pieces laid end to end and
// cut at even shares balance the workgroups better and took these chunks 222 us:
// parts of one sequence that begin at different keys read 711 MB past L2, not 278.)
constexpr size_t kWorkspaceCounters = 256 + kMaxRaggedSeqs * kKvHeads * 4;  // bytes of the words and counters
static_assert(kWorkspaceCounters % 256 == 0, "what lies behind is 256-byte aligned");
constexpr uint32_t kPackedPlanSeqs = 1024, kPackedLeastPart = 16, kPackedMaxParts = 400;
constexpr size_t kPackedPartPairs = 4 * 33 * 64;  // 4 waves x ((reference, sum), 64 outputs) x 64 lanes
struct PackedWorkspace {
    bool plan, narrow;
    uint32_t max_items, max_parts;
    size_t odd_offset, items_offset, arrived_offset, partials_offset, total;
};
inline PackedWorkspace packed_workspace_layout(uint32_t num_seqs, uint32_t rows, uint32_t max_context) {
    auto align = [](size_t v) { return (v + 255) / 256 * 256; };
    PackedWorkspace w{};
    w.narrow = packed_is_narrow(num_seqs, rows, max_context);
    w.plan = !w.narrow && num_seqs <= kPackedPlanSeqs;
    w.max_items = rows / kPackedTokens + num_seqs;
    if (w.plan && max_context > 32 * kPackedLeastPart) w.max_parts = kPackedMaxParts;
    w.max_items += w.max_parts;
    w.odd_offset = kWorkspaceCounters;
    w.items_offset = w.odd_offset + align((static_cast<size_t>(rows / kBlockTokens) + 2 * static_cast<size_t>(num_seqs)) * 4);
    w.arrived_offset = w.items_offset + align(w.plan ? w.max_items * sizeof(PackedItem) : 0);
    w.partials_offset = w.arrived_offset + align(w.max_parts * 2 * 4);
    w.total = w.partials_offset + static_cast<size_t>(w.max_parts) * 2 * kPackedPartPairs * 8;
    return w;
}

// A decode step of groups with shared pages (kernels_shared.hip).  ragged: the
// sequences, a row each.
constexpr int kSharedWaves = 4;
struct SharedRows {
    RaggedRows ragged;
    uint32_t num_groups, code;
    bool f32;
    const int32_t *group_offsets, *shared_lens;
    const void *query, *new_key, *new_value;
    void *out;
    const float *rope_cos, *rope_sin;
    uint32_t rope_rows;
    const int32_t *positions;
    uint32_t rotate_query;
    void *key_cache, *value_cache;
    uint8_t *exponents;
    float scale_log2;
    uint32_t *error_word;
    // sets of 2 * columns sequences, the parts that their shared rows and a
    // sequence's own are cut into, and what these leave for each kv head: outputs
    // [share][kv head][column][128] and (max in log2 units, sum) likewise, the
    // columns [shared part][columns * 16], then [sequence of the set][own part][8]
    uint32_t columns, shares, shared_parts, own_parts, unit_columns;
    float *part_o, *part_ml;
};
int launch_shared_decode(const SharedRows &rows, void *stream);
// Calls that the paged decode answers sooner, each sequence reading all of its
// rows: those of up to so many rows (num_seqs times max_context; what is shared,
// and how many rows there are, the host does not know), and those without a
// group of two.  Two launches take 11 us of any call, the paged decode's one 8:
// 4 sequences of 1221 rows 11.7 against 7.7 us (fp16) and 10.9 against 7.8 (e4m3), 16
// groups of 4 (80 thousand rows) 15.8 against 16.2 and 14.5 against 12.3, 12 groups
// of 8 (120 thousand) 16.3 against 20.4 and 15.9 against 18.9, 32 groups of 8 (320
// thousand) 26.8 against 44.4 and 25.5 against 31.7, 64 sequences with none in
// common 30.3 against 28.6 and 20.1 against 19.3.
constexpr uint32_t kSharedLeastRows = 90000;
inline bool shared_is_small(uint32_t num_seqs, uint32_t num_groups, uint32_t max_context, bool offsets) {
    if (num_seqs > kMaxRaggedSeqs || max_context > kMaxMergeParts * 4096) return false;
    return (!offsets && num_seqs == num_groups) || static_cast<uint64_t>(num_seqs) * max_context <= kSharedLeastRows;
}
// Its workspace: the paged decode's words and counters (0 the error word), which
// no call's parts lie on, then the parts' results.
constexpr uint32_t kMaxSharedSets = 16384;
struct SharedWorkspace {
    uint32_t columns, shares, shared_parts, own_parts, unit_columns;
    size_t part_o_offset, part_ml_offset, total;
};
inline SharedWorkspace shared_workspace_of(uint32_t columns, uint32_t shares, uint32_t max_context) {
    auto align = [](size_t v) { return (v + 255) / 256 * 256; };
    auto clamp = [](uint32_t v, uint32_t hi) { return v < 1 ? 1u : v > hi ? hi : v; };
    SharedWorkspace w{};
    w.columns = columns;
    w.shares = shares;
    const uint32_t most = clamp((max_context + 32 * kSharedWaves - 1) / (32 * kSharedWaves), 64);
    w.shared_parts = clamp((256 / (2 * w.shares) + 3) / 4 * 4, most);
    w.own_parts = clamp(128 / (2 * w.shares), most);
    w.unit_columns = w.shared_parts * w.columns * 16 + 2 * w.columns * w.own_parts * kGroup;
    const size_t all = static_cast<size_t>(w.shares) * 2 * w.unit_columns;
    w.part_o_offset = kWorkspaceCounters;
    w.part_ml_offset = w.part_o_offset + align(all * kHeadDim * 4);
    w.total = w.part_ml_offset + align(all * 8);
    return w;
}
inline SharedWorkspace shared_workspace_layout(uint32_t num_seqs, uint32_t num_groups, uint32_t max_context, bool offsets) {
    const uint32_t each = (num_seqs + num_groups - 1) / num_groups, columns = each <= 2 ? 1 : 2, set = 2 * columns;
    return shared_workspace_of(columns, offsets ? num_seqs / set + num_groups : num_groups * ((each + set - 1) / set), max_context);
}

// Prefill projection with fp16 weights: workspace of the exact hi/lo split
// of the activations ([rows][K] fp16 each) and the per-row exponents.
// Workspace of the projection: the hi/lo planes of the split activations in
// the GEMM's tile order -- for each 128-row tile t and each 32-wide k step s
// one 16 KiB block [plane (hi, lo)][k-chunk (4)][row (128)][8 fp16] -- then
// one exponent per row; rows are padded to a multiple of 128 (zeros).
constexpr uint32_t kProjectionTileRows = 128, kProjectionStepK = 32;
struct ProjectionWorkspace {
    uint16_t *tiles;
    int32_t *exponents;
};
struct ProjectionWorkspaceLayout {
    size_t exponents_offset, total;
};
inline ProjectionWorkspaceLayout projection_workspace_layout(uint32_t rows, uint32_t k_width) {
    const size_t padded = (static_cast<size_t>(rows) + kProjectionTileRows - 1) / kProjectionTileRows * kProjectionTileRows;
    const size_t tiles = padded * k_width * 4;  // two fp16 planes
    return {tiles, tiles + (padded * 4 + 255) / 256 * 256};
}
// The tiles of the projection GEMM (kernels_projection.hip), the threads of
// their workgroups, and the measured time of a compute unit's first tile and of
// each further one (0.1 us at a depth of 1024; medians over 24 numbers of rows
// from 8 to 4096 and ten pairs of widths, split kernel taken off), by preference
// on equal cost.  Two workgroups of the larger tiles overlap on a unit, the
// 512-thread group of 128 x 96 is alone there: its further tiles cost as much as
// those of 128 x 128.  (128 x 128's first is 169 by the median; 172 leaves q|k|v of
// 1025 to 1152 rows to two turns of 64 x 96, 1% faster for the layer.)
struct ProjectionTile {
    uint32_t rows, cols, threads, first, next;
};
constexpr ProjectionTile kProjectionTiles[] = {
    {128, 192, 256, 228, 210}, {128, 160, 256, 200, 168}, {128, 128, 256, 172, 138}, {128, 64, 512, 105, 92},
    {64, 64, 256, 82, 50},     {128, 96, 512, 134, 149},  {64, 96, 256, 101, 70},    {32, 64, 256, 66, 39},
    {16, 64, 256, 54, 28},     {16, 32, 512, 50, 21},     {16, 16, 512, 49, 14}};
constexpr int kProjectionTileCount = sizeof(kProjectionTiles) / sizeof(kProjectionTiles[0]);
constexpr uint32_t kXcds = 8;           // MI355X: 8 XCDs, each with its own L2
constexpr uint32_t kXcdUnits = 32;      // compute units of one XCD
constexpr uint32_t kXcdResident = 64;   // workgroups one XCD runs at once (two per compute unit)
struct ProjectionOrder {
    uint32_t row_tiles, col_tiles, col_groups, gen;
};

// Order of the tiles: the column grouping that gives the busiest compute unit
// the fewest tiles (the XCDs finish together), then the fewest operand bytes
// of an XCD's block (a row of activations is twice a row of weights), and
// generations of columns sized so that one generation is what an XCD runs at
// once.  *block receives the tiles of the largest block.  (The exact number of
// tiles in the first place cost bytes for nothing: 1600 rows, o 29.6 us against
// 26.7, down 37.1 against 34.7, four or eight column groups against one.)
inline ProjectionOrder projection_order(uint32_t row_tiles, uint32_t col_tiles, const ProjectionTile &t, uint64_t *block) {
    ProjectionOrder best{row_tiles, col_tiles, 1, 1};
    uint64_t best_turns = UINT64_MAX, best_bytes = UINT64_MAX;
    for (uint32_t gc = 1; gc <= kXcds; gc *= 2) {
        const uint32_t gr = kXcds / gc;
        const uint64_t rb = (row_tiles + gr - 1) / gr, cb = (col_tiles + gc - 1) / gc;
        const uint64_t turns = (rb * cb + kXcdUnits - 1) / kXcdUnits, bytes = rb * t.rows * 2 + cb * t.cols;
        if (turns < best_turns || (turns == best_turns && bytes < best_bytes)) {
            best_turns = turns;
            best_bytes = bytes;
            best.col_groups = gc;
            *block = rb * cb;
        }
    }
    const uint32_t gr = kXcds / best.col_groups, rb = (row_tiles + gr - 1) / gr;
    best.gen = kXcdResident / rb > 0 ? kXcdResident / rb : 1;
    return best;
}

// The tile of a launch: the least time of the busiest compute unit, which runs
// the tiles of the largest XCD block over the XCD's 32 units, by the measured
// times of its first tile and the further ones.  Against every tile timed at
// those rows and widths this picks the fastest or one within 6% of it, 0.2%
// slower on average.  (Clocks of the matrix or load path by the tile's area in
// place of measured times took 128 x 96 too often: 2500 rows of gate|up 87.3 us
// against 67.9 with 128 x 128, 3500 rows 117.5 against 88.7 with 128 x 192, 1836
// rows of 1152 to 4304 columns 55.4 against 46.7 with 128 x 160; where one turn
// does, that tile saves: 400 rows, gate|up 23.3 -> 20.9 us; 900 rows, q|k|v 23.5
// -> 20.8; 1157 rows, o 26.1 -> 24.0 and down 33.0 -> 30.4 with 64 x 96.)
// The grid, 8 times the largest block, keeps under 2^32 threads, which few rows
// of 2^30 or more columns exceed with the small tiles.  -1: no tile does.
inline int choose_projection_tile(uint32_t rows, uint32_t k_width, uint32_t n_width, ProjectionOrder *order, uint64_t *block) {
    int best = -1;
    uint64_t best_cost = UINT64_MAX;
    for (int i = 0; i < kProjectionTileCount; ++i) {
        const ProjectionTile t = kProjectionTiles[i];
        // The shifted last column tile needs a whole one, and a row of
        // weights at most 2^29 bytes (32-bit offsets over 8 rows); the 16 x 16
        // tile takes any.
        if (i + 1 < kProjectionTileCount && (n_width < t.cols || k_width > 1u << 28)) continue;
        uint64_t b = 0;
        const ProjectionOrder o = projection_order(rows / t.rows + (rows % t.rows != 0), n_width / t.cols + (n_width % t.cols != 0), t, &b);
        const uint64_t turns = (b + kXcdUnits - 1) / kXcdUnits, cost = t.first + (turns - 1) * t.next;
        if (cost < best_cost && b * kXcds * t.threads < 1ull << 32) {
            best_cost = cost;
            best = i;
            *order = o;
            *block = b;
        }
    }
    return best;
}

int launch_linear_projection_f16(const float *input, const uint16_t *weight, const float *bias, float *out,
                                 uint32_t rows, uint32_t k_width, uint32_t n_width, const ProjectionWorkspace &ws,
                                 void *stream);

// Split-K pair schedule of the causal prefill.  Query block qb (16 tokens)
// of one kv head attends qb/4 + 1 steps of 64 keys, so a grid of one
// workgroup per block is as long as its last block while most compute units
// idle.  With a workspace, block l and block qblocks-1-l of a kv head (about
// qblocks/4 + 2 steps together) go to two workgroups of about equal time:
// the first runs the first k steps of the heavy block, hands that part over,
// then runs the light block; the second runs the rest of the heavy block
// (which holds the diagonal) and merges the first part, which has arrived by
// then (otherwise the part that arrives last merges).  Running the heavy part
// first lets the second workgroup find it complete and merge it without
// storing its own part: config 4 at N=4096, 99.8-100.8 -> 96.6-97.3 us mean
// per call.  The workspace is asked for when the longest block is longer than
// kPrefillSplitSteps and used by prompts beyond kPrefillWaveTokens.  A pair
// whose light workgroup would take fewer than kPrefillSplitMin heavy steps at an even split is not
// split (the light block and the heavy block run whole on the two
// workgroups): a second segment costs its workgroup a query load, a pipeline
// fill and the partial hand-off, about what 4 to 5 steps cost (measured at
// N=4096: 9-13 us for 1-2 steps).  Of that, the light workgroup's extra
// segment (the one the heavy workgroup does not run: query load, fill, last
// steps and output stores of the light block) costs about 4 steps, so a
// split pair moves kPrefillSplitShift heavy steps from the light workgroup to
// the heavy one (config 4 at N=4096, shifts 0-3 on one box with the light
// block first: 103.0-103.7, 102.3, 100.0, 100.6-100.7 us mean per call; with
// the heavy part first, shifts 1-4: 97.7-97.9, 96.6-97.3, 97.6-98.8,
// 99.2-99.9).
constexpr uint32_t kPrefillSplitSteps = 32;
constexpr uint32_t kPrefillSplitMin = 5;
constexpr uint32_t kPrefillSplitShift = 2;
static_assert(kPrefillSplitMin > kPrefillSplitShift, "a split pair leaves the light workgroup a heavy step");
constexpr uint32_t kPrefillPartialFloats = 4 * 64 * 74;  // 4 waves x 64 lanes x (2 x 9 x 4 O/l + 2 m)

constexpr uint32_t prefill_block_steps(uint32_t qb) { return qb / 4 + 1; }
constexpr uint32_t prefill_max_steps(uint32_t qblocks) { return (qblocks - 1) / 4 + 1; }
constexpr uint32_t prefill_pairs(uint32_t qblocks) { return (qblocks + 1) / 2; }
// Longest prompt of prefill_wave_attention_kernel when the caller gave a
// workspace for the pair schedule (us, wave / pair: N=3000 f16 63.7 / 66.9,
// f32 77.6 / 83.0; 3500 80.2 / 75.0, 97.6 / 94.7; 4096 100.5 / 86.0, 124 /
// 112).  Shorter prompts still have a workspace size (from kPrefillSplitSteps
// on): callers compute, check and pass it, but nothing of it is touched.
constexpr uint32_t kPrefillWaveTokens = 3072;
static_assert(prefill_max_steps(kPrefillWaveTokens / 16 + 1) > kPrefillSplitSteps, "every paired prompt has a workspace");
constexpr uint32_t prefill_pair_workgroups(uint32_t qblocks) { return 4u * prefill_pairs(qblocks); }

struct PrefillSegment {
    uint32_t qb, part, nparts, step_begin, steps;
};

// Segments of workgroup w of the pair grid (w = (pair * 2 + g) * 2 + role);
// returns their number (0..2).
constexpr uint32_t prefill_pair_segments(uint32_t w, uint32_t qblocks, uint32_t *g, uint32_t *pair,
                                         PrefillSegment *first, PrefillSegment *second) {
    const uint32_t role = w & 1u, pg = w >> 1;
    *g = pg & 1u;
    *pair = pg >> 1;
    const uint32_t heavy = qblocks - 1u - *pair, light = *pair;
    const uint32_t sh = prefill_block_steps(heavy), sl = light == heavy ? 0u : prefill_block_steps(light);
    const uint32_t half = (sh - sl + 1u) / 2u;
    // heavy steps the light block's workgroup takes (>= 3 when split)
    const uint32_t k = half < kPrefillSplitMin ? 0u : half - kPrefillSplitShift;
    // Straight-line assignments (no runtime-indexed pointer), so that on the
    // device both segments stay in registers.  sh >= 1, so k >= sh implies k > 0.
    PrefillSegment s0{}, s1{};
    uint32_t n = 0;
    if (role == 0) {
        const PrefillSegment hs = k >= sh ? PrefillSegment{heavy, 0u, 1u, 0u, sh} : PrefillSegment{heavy, 0u, 2u, 0u, k};
        if (sl) {
            const PrefillSegment ls{light, 0u, 1u, 0u, sl};
            s0 = k > 0 ? hs : ls;  // the heavy part first, then the light block
            s1 = ls;
            n = k > 0 ? 2u : 1u;
        } else if (k > 0) {
            s0 = hs;
            n = 1;
        }
    } else if (k == 0) {
        s0 = {heavy, 0u, 1u, 0u, sh};
        n = 1;
    } else if (k < sh) {
        s0 = {heavy, 1u, 2u, k, sh - k};
        n = 1;
    }
    *first = s0;
    *second = s1;
    return n;
}
// Workspace of the pair schedule: an arrival counter per (pair, kv head),
// then two partial slabs each; 0 when the blocks are short enough.
struct PrefillWorkspace {
    size_t partial_offset, total;
};
inline PrefillWorkspace prefill_workspace_layout(uint32_t tokens) {
    const uint32_t qblocks = (tokens + 15u) / 16u;
    if (tokens == 0 || prefill_max_steps(qblocks) <= kPrefillSplitSteps) return {0, 0};
    const uint32_t items = 2u * prefill_pairs(qblocks);
    const size_t counters = (static_cast<size_t>(items) * 4 + 255) / 256 * 256;
    return {counters, counters + static_cast<size_t>(items) * 2 * kPrefillPartialFloats * 4};
}
int launch_gemv_f16(const uint16_t *weights, const float *vector, float *out, uint32_t rows, uint32_t columns,
                    void *stream);
constexpr uint32_t kGemvGroupMax = 4;
struct GemvGroup {  // members of one grouped GEMV launch (by value: kernel argument)
    const uint16_t *weights[kGemvGroupMax];
    float *out[kGemvGroupMax];
    uint32_t end[kGemvGroupMax - 1];  // rows up to the end of members 0..2; UINT32_MAX from the last member on
    uint32_t total;                   // rows of all members
};
int launch_gemv_group_f16(const GemvGroup &group, const float *vector, uint32_t columns, void *stream);

// Top-1 workspace: kTop1Slots slots of 256 bytes, each a packed u64
// candidate; zero before the first launch, zero again after each launch.
constexpr uint32_t kTop1Slots = 64;
struct Top1Slot {
    uint64_t best;
    uint64_t pad[31];
};
static_assert(sizeof(Top1Slot) == 256, "one slot per 256-byte line");
constexpr size_t kTop1WorkspaceBytes = kTop1Slots * sizeof(Top1Slot);
int launch_gemv_top1_f16(const uint16_t *weights, const float *vector, float *logits, uint32_t rows,
                         uint32_t columns, Top1Slot *slots, uint32_t *result, void *stream);
int launch_logits_top1_f32(const float *logits, uint32_t vocab, Top1Slot *slots, uint32_t *result, void *stream);

// Pages of a cache (kernels_pages.hip).  A page's part of a plane: block_bytes
// (a multiple of 4) at base + layer * layer_stride + id * block_bytes; `from`,
// where not null, is the other pool's plane that a copy reads.  wide: 16-byte
// accesses fit.
constexpr uint32_t kMaxPagePlanes = 4;
struct PagePlane {
    uint8_t *base;
    const uint8_t *from;
    uint64_t block_bytes, layer_stride;
    bool wide;
    uint64_t from_stride;
};
struct PagePlanes {
    PagePlane plane[kMaxPagePlanes];
    uint32_t count, layers;
};
// Rows of a fork (their plan is made in LDS).
constexpr uint32_t kMaxForkRows = 4096;
struct ForkRow {  // of the output: entries kept of the parent's, needed in all, its first fresh page, the page to copy to that (-1: none)
    int32_t parent;
    uint32_t kept, need, base;
    int32_t source;
    uint32_t length;
};
struct ForkInput {  // of the input: how many take it over, its filled blocks (shared by them), the end of what the first keeps
    uint32_t children, filled, kept, pad;
};
struct PagesFork {
    uint32_t num_blocks, max_blocks, rows_in, rows_out, appended, reserve_tokens, keep_inputs;
    const int32_t *tables_in, *lens_in, *parents, *reserve;
    int32_t *tables_out, *lens_out, *ref_counts;
    uint32_t *free_mask;
    struct {
        ForkRow *rows;
        ForkInput *inputs;
        int32_t *fresh;  // the pages taken, in order
        uint32_t *enough, *error_word;
    } plan;
};
struct PagesCompact {
    uint32_t num_blocks, max_blocks, rows;
    int32_t *tables, *forward, *ref_counts;
    uint32_t *free_mask;
    struct {
        uint32_t *used_before;     // by word of 32 pages, and the number in use behind them
        int32_t *from, *to, *rank;  // moves; a page's number among them, or -1
        uint32_t *moves;
    } plan;
};
// Workspace: 256 bytes of words (0 the error word, 1 whether a fork found its
// pages, 2 the moves of a compaction), then the plans' arrays; a fork's and a
// compaction's share theirs.
struct PagesWorkspace {
    size_t rows_offset, inputs_offset, first_offset, second_offset, third_offset, words_offset, total;
};
inline PagesWorkspace pages_workspace_layout(uint32_t num_blocks, uint32_t rows) {
    auto align = [](size_t v) { return (v + 255) / 256 * 256; };
    const size_t list = align(static_cast<size_t>(num_blocks) * 4);
    PagesWorkspace w{};
    w.rows_offset = 256;
    w.inputs_offset = w.rows_offset + align(static_cast<size_t>(rows) * sizeof(ForkRow));
    w.first_offset = w.inputs_offset + align(static_cast<size_t>(rows) * sizeof(ForkInput));
    w.second_offset = w.first_offset + list;
    w.third_offset = w.second_offset + list;
    w.words_offset = w.third_offset + list;
    w.total = w.words_offset + align((static_cast<size_t>(num_blocks) / 32 + 2) * 4);
    return w;
}
int launch_pages_reset(int32_t *refs, uint32_t *mask, uint32_t num_blocks, uint32_t *error_word, void *stream);
int launch_pages_fork(const PagesFork &f, const PagePlanes &planes, void *stream);
int launch_pages_compact(const PagesCompact &c, const PagePlanes &planes, void *stream);
int launch_pages_copy(const int32_t *src, const int32_t *dst, uint32_t count, uint32_t src_blocks, uint32_t dst_blocks, const PagePlanes &planes,
                      uint32_t *error_word, void *stream);

// Beam selection (kernels_beam.hip).  A row of logits is cut into segments of
// kBeamSegment; each leaves its best candidates as keys (logit and token in
// one number, see there) and its sum of exponentials.
constexpr uint32_t kBeamThreads = 256;
constexpr uint32_t kBeamMaxBeams = 64, kBeamMaxBest = 128;
// Logits a thread takes.  The same for any number of rows: what is summed
// together in f32 decides how a row's sum of exponentials is rounded, and a row's scores
// must not depend on what it is batched with.  (8 / 16 logits: four rows of 103424
// 10.5 / 10.5 us, one 9.0 / 8.7, four of 32000 10.7 / 10.2, 128 of 103424 27.7 / 22.4.)
constexpr uint32_t kBeamEach = 16, kBeamSegment = kBeamEach * kBeamThreads;
struct BeamSelect {
    uint32_t batch, beams, vocab, best, segments;
    uint64_t row_stride;
    const float *logits, *scores;
    const int32_t *finished;
    int32_t end_token;
    float *next_scores;
    int32_t *parents, *tokens, *next_finished;
    uint32_t *arrived;    // by batch entry: rows joined; the segments' launch clears them
    uint64_t *keys;       // [row][rank][segment]
    double *sums;         // [row][segment], relative to exp(reference)
    float *references;    // [row][segment]
    uint64_t *row_keys;   // [batch entry][rank][beam]: the scores' keys
    uint64_t *row_tokens;  // the same: token, and the score's f32 bits
};
struct BeamWorkspace {
    size_t keys_offset, sums_offset, references_offset, row_keys_offset, row_tokens_offset, total;
};
inline BeamWorkspace beam_workspace_layout(uint32_t batch, uint32_t beams, uint32_t vocab, uint32_t best) {
    auto align = [](size_t v) { return (v + 255) / 256 * 256; };
    const size_t rows = static_cast<size_t>(batch) * beams, parts = rows * ((static_cast<size_t>(vocab) + kBeamSegment - 1) / kBeamSegment);
    BeamWorkspace w{};
    w.keys_offset = align(static_cast<size_t>(batch) * 4);
    w.sums_offset = w.keys_offset + align(parts * best * 8);
    w.references_offset = w.sums_offset + align(parts * 8);
    w.row_keys_offset = w.references_offset + align(parts * 4);
    w.row_tokens_offset = w.row_keys_offset + align(rows * best * 8);
    w.total = w.row_tokens_offset + align(rows * best * 8);
    return w;
}
int launch_beam_select(const BeamSelect &b, void *stream);

// VisionPatchProjectionBytesDescriptor::plan (runtime-core lib.rs:1768-1840);
// returns a pvlc_hip_projection_error.
int32_t plan_projection(uint32_t patch_count, uint32_t input_width, uint32_t output_width, uint32_t weight_storage,
                        pvlc_hip_projection_plan *out);

// GemvTiledDescriptor::plan (runtime-core lib.rs:753-785); returns a status.
int plan_gemv_tiled(uint32_t rows, uint32_t columns, pvlc_hip_gemv_tiled_plan *out);

// Workspace layout of the paged decode.
struct DecodeWorkspace {
    size_t part_o_offset, part_ml_offset, counters_offset, error_offset, total;
    uint32_t part_stride;  // partials per (sequence, kv head) slot: max_parts rounded up to odd
};
DecodeWorkspace decode_workspace_layout(uint32_t num_seqs, uint32_t max_parts);
// Split-K state of one decode launch: partial outputs and (max, sum), merge
// counters (zero before the first launch; see kArrivalSpan), the error
// word and the two status words (automatic streaming partition, compute
// units).
struct DecodeState {
    float *part_o;
    float *part_ml;
    uint32_t *counters;
    uint32_t *error_word;
    uint32_t *status_words;
    uint32_t part_stride;  // partials per (sequence, kv head) slot: max_parts rounded up to odd
};
// Checks of pvlc_hip_paged_decode_f16's arguments, the workspace aside: the
// partition and the partitions per (sequence, kv head) of the launch.  With
// f32 operands (pvlc_hip_paged_decode_f32io) args' fp16 query, new key and
// value and output must be NULL and the f32 ones given.
pvlc_hip_status validate_decode_geometry(const pvlc_hip_paged_decode_args *a, uint32_t *partition_out,
                                         uint32_t *max_parts_out, const DecodeOperands32 *f32 = nullptr,
                                         bool codes = false);
// Launch a validated decode with its split-K state at `state`; launches_out
// receives the kernels launched (1, or 2 for the persistent kernel and its
// merge kernel).
pvlc_hip_status launch_decode_state(const pvlc_hip_paged_decode_args *a, uint32_t partition, uint32_t max_parts,
                                    const DecodeState &state, void *stream, uint32_t *launches_out,
                                    const DecodeOperands32 *f32 = nullptr, const DecodeCodes *codes = nullptr);
// The caller's workspace checked and laid out, then the launch; with codes the
// planes are 8-bit ones (passed through args' plane pointers).
pvlc_hip_status launch_decode_checked(const pvlc_hip_paged_decode_args *a, void *stream, uint32_t *launches_out = nullptr,
                                      const DecodeOperands32 *f32 = nullptr, const DecodeCodes *codes = nullptr);
// A HIP error as a status.
pvlc_hip_status hip_status(int error, const char *what);
// Partition rules: balanced_parts is the partition count per (sequence, kv
// head) of the single-shot rule; single_shot_partition returns 0 when a
// partition would exceed kSingleShotTiles; auto_partition falls back to
// 512-token (or longer) streaming partitions; auto_workspace_parts bounds the
// partitions of every automatic launch up to max_context.
uint32_t balanced_parts(uint32_t num_seqs);
uint32_t single_shot_partition(uint32_t num_seqs, uint32_t context);
uint32_t auto_partition(uint32_t num_seqs, uint32_t context);
uint32_t auto_workspace_parts(uint32_t num_seqs, uint32_t max_context);
// Launch shape for a partition: (waves, pairs) of the single-shot kernel,
// or of the persistent kernel when `streaming`.
struct DecodeShape {
    uint32_t waves, pairs;
};
DecodeShape decode_shape(uint32_t partition_tokens, bool streaming);

}  // namespace pvlc
