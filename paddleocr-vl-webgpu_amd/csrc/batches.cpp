// Entry points of batches over paged caches (appends of several sequences' rows,
// packed prompts, decode with shared pages): argument checks before any GPU effect, then the launches.

#include <cstdint>
#include <initializer_list>
#include <string>

#include "pvlc_internal.hpp"

using namespace pvlc;

namespace {

constexpr uint64_t kMaxGroups = 1u << 24;  // workgroups of 256 threads that a launch may have (below 2^32 threads)
constexpr uint64_t kMaxStride = 1ull << 31;
constexpr uint32_t kMaxTokens = 0x7FFFFF00u;  // of a table's row: positions rounded up to a few blocks stay whole numbers of 32 bits

bool aligned(const void *p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

struct Range {
    const void *at;
    uint64_t bytes;
};

bool overlap(const Range &a, const Range &b) {
    const auto x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
    return a.at && b.at && a.bytes && b.bytes && x < y + b.bytes && y < x + a.bytes;
}

pvlc_hip_status check_planes(uint32_t code, const void *keys, const void *values, const void *exponents) {
    if (code != PVLC_HIP_KV_F16 && code != PVLC_HIP_KV_E4M3 && code != PVLC_HIP_KV_INT8)
        return invalid(PVLC_HIP_INV_INVALID_ACTIVATION_LAYOUT,
                       "the cache's code is PVLC_HIP_KV_F16, PVLC_HIP_KV_E4M3 or PVLC_HIP_KV_INT8, not " + std::to_string(code));
    if (!keys || !values || (code != PVLC_HIP_KV_F16 && !exponents))
        return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "cache plane or exponents pointer is NULL");
    if (!aligned(keys, 16) || !aligned(values, 16) || (code != PVLC_HIP_KV_F16 && !aligned(exponents, 4)))
        return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "cache planes must be 16-byte aligned, exponents 4-byte aligned");
    return PVLC_HIP_OK;
}

// A matrix of `rows` rows of `width` elements, `stride` (0: width) apart.
pvlc_hip_status check_matrix(const void *at, uint64_t *stride, uint32_t rows, uint32_t width, uint32_t size, const char *name, Range *range) {
    if (!at) return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, std::string(name) + " pointer is NULL");
    if (!aligned(at, 16)) return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, std::string(name) + " must be 16-byte aligned");
    if (*stride == 0) *stride = width;
    if (*stride < width || *stride >= kMaxStride || *stride * size % 16 != 0)
        return invalid(PVLC_HIP_INV_INVALID_ACTIVATION_LAYOUT,
                       std::string(name) + " rows must lie apart, a multiple of 16 bytes and below 2^31 elements from one to the next");
    *range = {at, ((rows - 1) * *stride + width) * size};
    return PVLC_HIP_OK;
}

// An append's arguments, the overlaps aside, as the kernels take them.
pvlc_hip_status check_append(const pvlc_hip_kv_append_args *args, const void *key, const void *value, bool f32, AppendRows *out, Range *keys,
                             Range *values) {
    if (pvlc_hip_status st = check_planes(args->code, args->key_cache, args->value_cache, args->exponents)) return st;
    if (args->num_seqs == 0 || args->rows == 0 || args->num_blocks == 0 || args->max_blocks_per_seq == 0)
        return invalid(PVLC_HIP_INV_ZERO_DIMENSION, "sequences, rows, blocks and table width must be nonzero");
    if (args->rows > 0x7FFFFFFFu || args->num_blocks > 0x7FFFFFFFu || args->max_blocks_per_seq > kMaxTokens / kBlockTokens)
        return invalid(PVLC_HIP_INV_INVALID_DECODER_GEOMETRY, "rows and blocks must be below 2^31, a table row's tokens up to 2^31 - 256");
    if (args->rows / kBlockTokens + 2ull * args->num_seqs >= kMaxGroups)
        return invalid(PVLC_HIP_INV_INVALID_DECODER_GEOMETRY, "rows and sequences exceed the grid");
    if (!args->row_offsets && args->rows % args->num_seqs != 0)
        return invalid(PVLC_HIP_INV_INVALID_SEQUENCE_BOUNDARIES, "without offsets the rows must divide among the sequences");
    if (!args->block_tables && static_cast<uint64_t>(args->num_seqs) * args->max_blocks_per_seq > args->num_blocks)
        return invalid(PVLC_HIP_INV_INVALID_DECODER_GEOMETRY, "the sequences' contiguous blocks exceed the planes");
    for (const void *p : {static_cast<const void *>(args->row_offsets), static_cast<const void *>(args->block_tables),
                          static_cast<const void *>(args->cache_lens), static_cast<const void *>(args->positions),
                          static_cast<const void *>(args->error_word)})
        if (!aligned(p, 4)) return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "offsets, tables, lengths, positions and error word must be 4-byte aligned");
    if ((args->rope_cos == nullptr) != (args->rope_sin == nullptr) || (args->rope_cos && args->rope_rows == 0))
        return invalid(PVLC_HIP_INV_INVALID_ROTARY_DIMENSION, "rotary tables must be given together with rows");
    if (!aligned(args->rope_cos, 16) || !aligned(args->rope_sin, 16))
        return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "rotary tables must be 16-byte aligned");
    const uint32_t size = f32 ? 4 : 2;
    uint64_t key_stride = args->key_stride, value_stride = args->value_stride;
    if (pvlc_hip_status st = check_matrix(key, &key_stride, args->rows, kRowElems, size, "key", keys)) return st;
    if (pvlc_hip_status st = check_matrix(value, &value_stride, args->rows, kRowElems, size, "value", values)) return st;
    *out = {};
    out->ragged = {args->num_seqs, args->rows, args->rows / args->num_seqs, args->row_offsets, args->cache_lens, args->num_blocks,
                   args->max_blocks_per_seq, args->block_tables, args->max_blocks_per_seq * kBlockTokens};
    out->code = args->code;
    out->f32 = f32;
    out->key = key;
    out->value = value;
    out->key_stride = static_cast<int64_t>(key_stride);
    out->value_stride = static_cast<int64_t>(value_stride);
    out->rope_cos = args->rope_cos;
    out->rope_sin = args->rope_sin;
    out->rope_rows = args->rope_rows;
    out->positions = args->positions;
    out->key_cache = args->key_cache;
    out->value_cache = args->value_cache;
    out->exponents = args->exponents;
    out->error_word = args->error_word;
    return PVLC_HIP_OK;
}

// What the call writes lies apart from what it reads and from one another.
pvlc_hip_status check_apart(const pvlc_hip_kv_append_args &a, const Range &keys, const Range &values, std::initializer_list<Range> reads,
                            std::initializer_list<Range> writes) {
    const uint64_t plane = static_cast<uint64_t>(a.num_blocks) * kKvHeads * kBlockHeadElems * (a.code == PVLC_HIP_KV_F16 ? 2 : 1);
    Range read[16] = {keys, values,
                      {a.row_offsets, 4ull * a.num_seqs + 4},
                      {a.block_tables, 4ull * a.num_seqs * a.max_blocks_per_seq},
                      {a.cache_lens, 4ull * a.num_seqs},
                      {a.positions, 4ull * a.rows},
                      {a.rope_cos, 256ull * a.rope_rows},
                      {a.rope_sin, 256ull * a.rope_rows}};
    Range written[8] = {{a.key_cache, plane}, {a.value_cache, plane}, {a.code == PVLC_HIP_KV_F16 ? nullptr : a.exponents, 4ull * a.num_blocks}};
    int n = 8, m = 3;
    for (const Range &r : reads) read[n++] = r;
    for (const Range &r : writes) written[m++] = r;
    for (int w = 0; w < m; ++w) {
        for (int r = 0; r < n; ++r)
            if (overlap(written[w], read[r]))
                return invalid(PVLC_HIP_INV_INVALID_ACTIVATION_LAYOUT, "planes, exponents, workspace and output may not overlap the call's inputs");
        for (int v = 0; v < w; ++v)
            if (overlap(written[w], written[v]))
                return invalid(PVLC_HIP_INV_INVALID_ACTIVATION_LAYOUT, "planes, exponents, workspace and output may not overlap");
    }
    return PVLC_HIP_OK;
}

template <class Args>
pvlc_hip_status check_context(const Args *a) {
    if (a->max_context == 0) return invalid(PVLC_HIP_INV_ZERO_DIMENSION, "max_context must be nonzero");
    if (a->max_context > static_cast<uint64_t>(a->max_blocks_per_seq) * kBlockTokens)
        return invalid(PVLC_HIP_INV_INVALID_DECODER_GEOMETRY, "max_context exceeds a sequence's table");
    return PVLC_HIP_OK;
}

template <class Args>
pvlc_hip_status check_workspace(const Args *a, size_t bytes, const char *what) {
    if (!a->workspace || !aligned(a->workspace, 256))
        return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, std::string(what) + " workspace must be given, 256-byte aligned");
    if (a->workspace_bytes < bytes)
        return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, std::string(what) + " workspace holds " + std::to_string(a->workspace_bytes) +
                                                         " bytes but the call needs " + std::to_string(bytes));
    return PVLC_HIP_OK;
}

pvlc_hip_status append(const pvlc_hip_kv_append_args *args, const void *key, const void *value, bool f32, void *stream) {
    if (!args) return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "append args are NULL");
    AppendRows a{};
    Range keys, values;
    if (pvlc_hip_status st = check_append(args, key, value, f32, &a, &keys, &values)) return st;
    if (pvlc_hip_status st = check_apart(*args, keys, values, {}, {{args->error_word, 4}})) return st;
    if (const int e = launch_kv_append(a, stream)) return hip_status(e, "append launch");
    return ok();
}

pvlc_hip_status prefill(const pvlc_hip_packed_prefill_args *args, const void *query, const void *key, const void *value, void *out, bool f32,
                        void *stream) {
    if (!args) return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "packed prefill args are NULL");
    pvlc_hip_kv_append_args rows{};
    rows.num_seqs = args->num_seqs;
    rows.rows = args->rows;
    rows.num_blocks = args->num_blocks;
    rows.max_blocks_per_seq = args->max_blocks_per_seq;
    rows.code = PVLC_HIP_KV_F16;
    rows.row_offsets = args->row_offsets;
    rows.block_tables = args->block_tables;
    rows.cache_lens = args->cache_lens;
    rows.key_cache = args->key_cache;
    rows.value_cache = args->value_cache;
    rows.key_stride = args->key_stride;
    rows.value_stride = args->value_stride;
    rows.rope_cos = args->rope_cos;
    rows.rope_sin = args->rope_sin;
    rows.rope_rows = args->rope_rows;
    rows.positions = args->positions;
    rows.error_word = static_cast<uint32_t *>(args->workspace);
    AppendRows a{};
    Range keys, values;
    if (pvlc_hip_status st = check_append(&rows, key, value, f32, &a, &keys, &values)) return st;
    if (pvlc_hip_status st = check_context(args)) return st;
    const uint32_t size = f32 ? 4 : 2;
    uint64_t query_stride = args->query_stride, out_stride = 0;
    Range queries, outs;
    if (pvlc_hip_status st = check_matrix(query, &query_stride, args->rows, kQueryHeads * kHeadDim, size, "query", &queries)) return st;
    if (pvlc_hip_status st = check_matrix(out, &out_stride, args->rows, kQueryHeads * kHeadDim, size, "out", &outs)) return st;
    const PackedWorkspace ws = packed_workspace_layout(args->num_seqs, args->rows, args->max_context);
    if (2ull * ws.max_items >= kMaxGroups)
        return invalid(PVLC_HIP_INV_INVALID_DECODER_GEOMETRY, "rows and sequences of a packed prefill exceed the grid");
    if (pvlc_hip_status st = check_workspace(args, ws.total, "packed prefill")) return st;
    if (pvlc_hip_status st = check_apart(rows, keys, values, {queries}, {{args->workspace, ws.total}, outs})) return st;
    a.ragged.max_tokens = args->max_context;
    PackedRows r{};
    r.ragged = a.ragged;
    r.f32 = f32;
    r.query = query;
    r.out = out;
    r.query_stride = static_cast<int64_t>(query_stride);
    r.rope_cos = args->rope_cos;
    r.rope_sin = args->rope_sin;
    r.rope_rows = args->rope_rows;
    r.positions = args->positions;
    r.key_cache = args->key_cache;
    r.value_cache = args->value_cache;
    r.error_word = a.error_word;
    auto *base = static_cast<unsigned char *>(args->workspace);
    if (ws.plan) {
        a.plan.count = reinterpret_cast<int32_t *>(base) + 1;
        a.plan.items = reinterpret_cast<PackedItem *>(base + ws.items_offset);
        a.plan.arrived = reinterpret_cast<uint32_t *>(base + ws.arrived_offset);
        a.plan.max_items = ws.max_items;
        a.plan.max_parts = ws.max_parts;
    }
    a.odd = reinterpret_cast<uint32_t *>(base + ws.odd_offset);
    r.odd = reinterpret_cast<const int32_t *>(a.odd);
    r.count = a.plan.count;
    r.items = a.plan.items;
    r.arrived = a.plan.arrived;
    r.partials = reinterpret_cast<uint64_t *>(base + ws.partials_offset);
    r.narrow = ws.narrow;
    r.max_items = ws.max_items;
    if (const int e = launch_kv_append(a, stream)) return hip_status(e, "packed prefill append launch");
    if (const int e = launch_packed_prefill(r, stream)) return hip_status(e, "packed prefill launch");
    return ok();
}

// The call as a paged decode (its checks are those of that one's arguments).
pvlc_hip_status decode_alone(const pvlc_hip_shared_decode_args *args, const void *query, const void *key, const void *value, void *out, bool f32,
                             void *stream) {
    pvlc_hip_paged_decode_args d{};
    d.num_seqs = args->num_seqs;
    d.num_blocks = args->num_blocks;
    d.max_blocks_per_seq = args->max_blocks_per_seq;
    d.block_tables = args->block_tables;
    d.cache_lens = args->cache_lens;
    d.max_context = args->max_context;
    d.key_cache = static_cast<uint16_t *>(args->key_cache);
    d.value_cache = static_cast<uint16_t *>(args->value_cache);
    d.rope_cos = args->rope_cos;
    d.rope_sin = args->rope_sin;
    d.rope_rows = args->rope_rows;
    d.positions = args->positions;
    d.rotate_query = args->rotate_query;
    d.workspace = args->workspace;
    d.workspace_bytes = args->workspace_bytes;
    DecodeOperands32 o{};
    if (f32) {
        o = {static_cast<const float *>(query), static_cast<const float *>(key), static_cast<const float *>(value), static_cast<float *>(out)};
    } else {
        d.query = static_cast<const uint16_t *>(query);
        d.new_key = static_cast<const uint16_t *>(key);
        d.new_value = static_cast<const uint16_t *>(value);
        d.out = static_cast<uint16_t *>(out);
    }
    const DecodeCodes codes{args->code, args->exponents};
    if (pvlc_hip_status st = launch_decode_checked(&d, stream, nullptr, f32 ? &o : nullptr, args->code == PVLC_HIP_KV_F16 ? nullptr : &codes)) return st;
    return ok();
}

// The most that a shared decode of up to so many sequences, groups and rows needs.
// It is not what the largest one needs: fewer sets are cut into more parts, and
// fewer sequences may run as paged decodes, whose parts are others.
size_t most_shared_bytes(uint32_t num_seqs, uint32_t num_groups, uint32_t max_context) {
    size_t most = 0;
    auto take = [&](size_t bytes) { most = bytes > most ? bytes : most; };
    for (uint32_t columns = 1; columns <= 2; ++columns) {
        const uint64_t sets = static_cast<uint64_t>(num_seqs) / (2 * columns) + num_groups;  // of a call of any offsets, or none, at most
        const uint32_t shares = static_cast<uint32_t>(sets < kMaxSharedSets ? sets : kMaxSharedSets);
        // (of more than 256 sets all have one part of either kind)
        for (uint32_t n = 1; n <= shares && n <= 256; ++n) take(shared_workspace_of(columns, n, max_context).total);
        take(shared_workspace_of(columns, shares, max_context).total);
    }
    for (uint32_t n = 1; n <= num_seqs && n <= kMaxRaggedSeqs; ++n) {
        // The longest context that n sequences may run alone with; they are cut
        // into balanced_parts, or from 512 rows on.
        uint32_t rows = n <= num_groups ? max_context : kSharedLeastRows / n;
        rows = rows < max_context ? rows : max_context;
        const uint32_t cut = rows / 512 + 1, parts = balanced_parts(n), streamed = cut < kMaxMergeParts ? cut : kMaxMergeParts;
        if (rows > 0) take(decode_workspace_layout(n, parts > streamed ? parts : streamed).total);
    }
    return most;
}

pvlc_hip_status shared(const pvlc_hip_shared_decode_args *args, const void *query, const void *key, const void *value, void *out, bool f32,
                       void *stream) {
    if (!args) return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "shared decode args are NULL");
    if (args->num_groups == 0) return invalid(PVLC_HIP_INV_ZERO_DIMENSION, "groups must be nonzero");
    if (!args->block_tables || !args->cache_lens || !args->shared_lens)
        return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "shared decode tables, lengths and shared lengths must be given");
    pvlc_hip_kv_append_args rows{};
    rows.num_seqs = rows.rows = args->num_seqs;
    rows.num_blocks = args->num_blocks;
    rows.max_blocks_per_seq = args->max_blocks_per_seq;
    rows.code = args->code;
    rows.block_tables = args->block_tables;
    rows.cache_lens = args->cache_lens;
    rows.key_cache = args->key_cache;
    rows.value_cache = args->value_cache;
    rows.exponents = args->exponents;
    rows.rope_cos = args->rope_cos;
    rows.rope_sin = args->rope_sin;
    rows.rope_rows = args->rope_rows;
    rows.positions = args->positions;
    rows.error_word = static_cast<uint32_t *>(args->workspace);
    AppendRows a{};
    Range keys, values;
    if (pvlc_hip_status st = check_append(&rows, key, value, f32, &a, &keys, &values)) return st;
    if (!args->group_offsets && args->num_seqs % args->num_groups != 0)
        return invalid(PVLC_HIP_INV_INVALID_SEQUENCE_BOUNDARIES, "without offsets the sequences must divide among the groups");
    if (static_cast<uint64_t>(args->num_seqs) + args->num_groups > kMaxSharedSets)
        return invalid(PVLC_HIP_INV_INVALID_DECODER_GEOMETRY, "sequences and groups of a shared decode exceed 16384");
    if (!aligned(args->group_offsets, 4) || !aligned(args->shared_lens, 4))
        return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "group offsets and shared lengths must be 4-byte aligned");
    if (pvlc_hip_status st = check_context(args)) return st;
    const uint32_t size = f32 ? 4 : 2;
    uint64_t query_stride = 0, out_stride = 0;
    Range queries, outs;
    if (pvlc_hip_status st = check_matrix(query, &query_stride, args->num_seqs, kQueryHeads * kHeadDim, size, "query", &queries)) return st;
    if (pvlc_hip_status st = check_matrix(out, &out_stride, args->num_seqs, kQueryHeads * kHeadDim, size, "out", &outs)) return st;
    const bool offsets = args->group_offsets != nullptr;
    const bool small = shared_is_small(args->num_seqs, args->num_groups, args->max_context, offsets);
    const SharedWorkspace ws = shared_workspace_layout(args->num_seqs, args->num_groups, args->max_context, offsets);
    const size_t needed = small ? pvlc_hip_paged_decode_workspace_bytes(args->num_seqs, args->max_context, 0) : ws.total;
    if (pvlc_hip_status st = check_workspace(args, needed, "shared decode")) return st;
    const Range groups{args->group_offsets, 4ull * args->num_groups + 4}, lens{args->shared_lens, 4ull * args->num_groups};
    if (pvlc_hip_status st = check_apart(rows, keys, values, {queries, groups, lens}, {{args->workspace, needed}, outs})) return st;
    if (small) return decode_alone(args, query, key, value, out, f32, stream);
    a.ragged.max_tokens = args->max_context;
    auto *base = static_cast<unsigned char *>(args->workspace);
    SharedRows r{};
    r.ragged = a.ragged;
    r.num_groups = args->num_groups;
    r.code = args->code;
    r.f32 = f32;
    r.group_offsets = args->group_offsets;
    r.shared_lens = args->shared_lens;
    r.query = query;
    r.new_key = key;
    r.new_value = value;
    r.out = out;
    r.rope_cos = args->rope_cos;
    r.rope_sin = args->rope_sin;
    r.rope_rows = args->rope_rows;
    r.positions = args->positions;
    r.rotate_query = args->rotate_query;
    r.key_cache = args->key_cache;
    r.value_cache = args->value_cache;
    r.exponents = args->exponents;
    r.error_word = a.error_word;
    r.columns = ws.columns;
    r.shares = ws.shares;
    r.shared_parts = ws.shared_parts;
    r.own_parts = ws.own_parts;
    r.unit_columns = ws.unit_columns;
    r.part_o = reinterpret_cast<float *>(base + ws.part_o_offset);
    r.part_ml = reinterpret_cast<float *>(base + ws.part_ml_offset);
    if (const int e = launch_shared_decode(r, stream)) return hip_status(e, "shared decode launch");
    return ok();
}

}  // namespace

extern "C" {

pvlc_hip_status pvlc_hip_kv_append_f16(const pvlc_hip_kv_append_args *args, const uint16_t *key, const uint16_t *value, void *stream) {
    return append(args, key, value, false, stream);
}

pvlc_hip_status pvlc_hip_kv_append_f32(const pvlc_hip_kv_append_args *args, const float *key, const float *value, void *stream) {
    return append(args, key, value, true, stream);
}

size_t pvlc_hip_packed_prefill_workspace_bytes(uint32_t num_seqs, uint32_t rows, uint32_t max_context) {
    if (num_seqs == 0 || rows == 0 || max_context == 0) return 0;
    // (past kPackedPlanSeqs sequences a call has no plan, and no parts; a smaller one has both)
    const size_t own = packed_workspace_layout(num_seqs, rows, max_context).total;
    const size_t planned = packed_workspace_layout(num_seqs < kPackedPlanSeqs ? num_seqs : kPackedPlanSeqs, rows, max_context).total;
    return own > planned ? own : planned;
}

pvlc_hip_status pvlc_hip_packed_prefill_f16(const pvlc_hip_packed_prefill_args *args, const uint16_t *query, const uint16_t *key,
                                            const uint16_t *value, uint16_t *out, void *stream) {
    return prefill(args, query, key, value, out, false, stream);
}

pvlc_hip_status pvlc_hip_packed_prefill_f32io(const pvlc_hip_packed_prefill_args *args, const float *query, const float *key,
                                              const float *value, float *out, void *stream) {
    return prefill(args, query, key, value, out, true, stream);
}

size_t pvlc_hip_shared_decode_workspace_bytes(uint32_t num_seqs, uint32_t num_groups, uint32_t max_context) {
    if (num_seqs == 0 || num_groups == 0 || max_context == 0) return 0;
    return most_shared_bytes(num_seqs, num_groups, max_context);
}

pvlc_hip_status pvlc_hip_shared_decode_f16(const pvlc_hip_shared_decode_args *args, const uint16_t *query, const uint16_t *new_key,
                                           const uint16_t *new_value, uint16_t *out, void *stream) {
    return shared(args, query, new_key, new_value, out, false, stream);
}

pvlc_hip_status pvlc_hip_shared_decode_f32io(const pvlc_hip_shared_decode_args *args, const float *query, const float *new_key,
                                             const float *new_value, float *out, void *stream) {
    return shared(args, query, new_key, new_value, out, true, stream);
}

}  // extern "C"
