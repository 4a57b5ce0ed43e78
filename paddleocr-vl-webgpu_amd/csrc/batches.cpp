// Entry points of batches over paged caches (appends of several sequences' rows,
// packed prompts): argument checks before any GPU effect, then the launches.

#include <cstdint>
#include <initializer_list>
#include <string>

#include "pvlc_internal.hpp"

using namespace pvlc;

namespace {

constexpr uint64_t kMaxGroups = 1u << 24;  // workgroups of 256 threads that a launch may have (below 2^32 threads)
constexpr uint64_t kMaxStride = 1ull << 31;

bool aligned(const void *p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

struct Range {
    const void *at;
    uint64_t bytes;
};

bool overlap(const Range &a, const Range &b) {
    const auto x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
    return a.at && b.at && a.bytes && b.bytes && x < y + b.bytes && y < x + a.bytes;
}

pvlc_hip_status apart(std::initializer_list<Range> written, std::initializer_list<Range> read, const char *what) {
    for (const Range *w = written.begin(); w != written.end(); ++w) {
        for (const Range &r : read)
            if (overlap(*w, r)) return invalid(PVLC_HIP_INV_INVALID_ACTIVATION_LAYOUT, std::string(what) + " overlap its inputs");
        for (const Range *v = written.begin(); v != w; ++v)
            if (overlap(*w, *v)) return invalid(PVLC_HIP_INV_INVALID_ACTIVATION_LAYOUT, std::string(what) + " overlap one another");
    }
    return PVLC_HIP_OK;
}

// What the calls of this file have in common.
template <class Args>
pvlc_hip_status check_rows(const Args *a, uint32_t share, uint32_t spare) {
    if (a->num_seqs == 0 || a->rows == 0 || a->num_blocks == 0 || a->max_blocks_per_seq == 0)
        return invalid(PVLC_HIP_INV_ZERO_DIMENSION, "sequences, rows, blocks and table width must be nonzero");
    if (a->rows > 0x7FFFFFFFu || a->num_blocks > 0x7FFFFFFFu || a->max_blocks_per_seq > 0x7FFFFFFFu / kBlockTokens)
        return invalid(PVLC_HIP_INV_INVALID_DECODER_GEOMETRY, "rows, blocks and a table row's tokens must be below 2^31");
    if (a->rows / share + static_cast<uint64_t>(spare) * a->num_seqs >= kMaxGroups)
        return invalid(PVLC_HIP_INV_INVALID_DECODER_GEOMETRY, "rows and sequences exceed the grid");
    if (!a->row_offsets && a->rows % a->num_seqs != 0)
        return invalid(PVLC_HIP_INV_INVALID_SEQUENCE_BOUNDARIES, "without offsets the rows must divide among the sequences");
    if (!a->block_tables && static_cast<uint64_t>(a->num_seqs) * a->max_blocks_per_seq > a->num_blocks)
        return invalid(PVLC_HIP_INV_INVALID_DECODER_GEOMETRY, "the sequences' contiguous blocks exceed the planes");
    for (const void *p : {static_cast<const void *>(a->row_offsets), static_cast<const void *>(a->block_tables),
                          static_cast<const void *>(a->cache_lens), static_cast<const void *>(a->positions)})
        if (!aligned(p, 4)) return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "offsets, tables, lengths and positions must be 4-byte aligned");
    return PVLC_HIP_OK;
}

template <class Args>
pvlc_hip_status check_rope(const Args *a) {
    if ((a->rope_cos == nullptr) != (a->rope_sin == nullptr) || (a->rope_cos && a->rope_rows == 0))
        return invalid(PVLC_HIP_INV_INVALID_ROTARY_DIMENSION, "rotary tables must be given together with rows");
    if (!aligned(a->rope_cos, 16) || !aligned(a->rope_sin, 16))
        return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "rotary tables must be 16-byte aligned");
    return PVLC_HIP_OK;
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

uint64_t plane_bytes(uint32_t num_blocks, uint32_t code) {
    return static_cast<uint64_t>(num_blocks) * kKvHeads * kBlockHeadElems * (code == PVLC_HIP_KV_F16 ? 2 : 1);
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

template <class Args>
RaggedRows ragged_rows(const Args *a) {
    return {a->num_seqs, a->rows, a->rows / a->num_seqs, a->row_offsets, a->cache_lens, a->num_blocks, a->max_blocks_per_seq, a->block_tables,
            a->max_blocks_per_seq * kBlockTokens};
}

pvlc_hip_status append(const pvlc_hip_kv_append_args *args, const void *key, const void *value, bool f32, void *stream) {
    if (!args) return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "append args are NULL");
    if (pvlc_hip_status st = check_planes(args->code, args->key_cache, args->value_cache, args->exponents)) return st;
    if (pvlc_hip_status st = check_rows(args, kBlockTokens, 2)) return st;
    if (pvlc_hip_status st = check_rope(args)) return st;
    if (!aligned(args->error_word, 4)) return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "the error word must be 4-byte aligned");
    const uint32_t size = f32 ? 4 : 2;
    uint64_t key_stride = args->key_stride, value_stride = args->value_stride;
    Range keys, values;
    if (pvlc_hip_status st = check_matrix(key, &key_stride, args->rows, kRowElems, size, "key", &keys)) return st;
    if (pvlc_hip_status st = check_matrix(value, &value_stride, args->rows, kRowElems, size, "value", &values)) return st;
    const uint64_t bytes = plane_bytes(args->num_blocks, args->code);
    const bool codes = args->code != PVLC_HIP_KV_F16;
    if (pvlc_hip_status st = apart({{args->key_cache, bytes},
                                    {args->value_cache, bytes},
                                    {codes ? args->exponents : nullptr, 4ull * args->num_blocks},
                                    {args->error_word, 4}},
                                   {keys, values,
                                    {args->row_offsets, 4ull * args->num_seqs + 4},
                                    {args->block_tables, 4ull * args->num_seqs * args->max_blocks_per_seq},
                                    {args->cache_lens, 4ull * args->num_seqs},
                                    {args->positions, 4ull * args->rows},
                                    {args->rope_cos, 256ull * args->rope_rows},
                                    {args->rope_sin, 256ull * args->rope_rows}},
                                   "an append's planes, exponents and error word"))
        return st;
    AppendRows a{};
    a.ragged = ragged_rows(args);
    a.code = args->code;
    a.f32 = f32;
    a.key = key;
    a.value = value;
    a.key_stride = static_cast<int64_t>(key_stride);
    a.value_stride = static_cast<int64_t>(value_stride);
    a.rope_cos = args->rope_cos;
    a.rope_sin = args->rope_sin;
    a.rope_rows = args->rope_rows;
    a.positions = args->positions;
    a.key_cache = args->key_cache;
    a.value_cache = args->value_cache;
    a.exponents = args->exponents;
    a.error_word = args->error_word;
    const int e = launch_kv_append(a, stream);
    if (e != 0) return hip_status(e, "append launch");
    return ok();
}

pvlc_hip_status prefill(const pvlc_hip_packed_prefill_args *args, const void *query, const void *key, const void *value, void *out, bool f32,
                        void *stream) {
    if (!args) return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "packed prefill args are NULL");
    if (pvlc_hip_status st = check_planes(PVLC_HIP_KV_F16, args->key_cache, args->value_cache, nullptr)) return st;
    if (pvlc_hip_status st = check_rows(args, kBlockTokens, 2)) return st;
    if (pvlc_hip_status st = check_rope(args)) return st;
    if (args->max_context == 0) return invalid(PVLC_HIP_INV_ZERO_DIMENSION, "max_context must be nonzero");
    if (args->max_context > static_cast<uint64_t>(args->max_blocks_per_seq) * kBlockTokens)
        return invalid(PVLC_HIP_INV_INVALID_DECODER_GEOMETRY, "max_context exceeds a sequence's table");
    const uint32_t size = f32 ? 4 : 2;
    uint64_t query_stride = args->query_stride, key_stride = args->key_stride, value_stride = args->value_stride, out_stride = 0;
    Range queries, keys, values, outs;
    if (pvlc_hip_status st = check_matrix(query, &query_stride, args->rows, kQueryHeads * kHeadDim, size, "query", &queries)) return st;
    if (pvlc_hip_status st = check_matrix(key, &key_stride, args->rows, kRowElems, size, "key", &keys)) return st;
    if (pvlc_hip_status st = check_matrix(value, &value_stride, args->rows, kRowElems, size, "value", &values)) return st;
    if (pvlc_hip_status st = check_matrix(out, &out_stride, args->rows, kQueryHeads * kHeadDim, size, "out", &outs)) return st;
    const PackedWorkspace ws = packed_workspace_layout(args->num_seqs, args->rows, args->max_context);
    if (!args->workspace || !aligned(args->workspace, 256))
        return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "packed prefill workspace must be given, 256-byte aligned");
    if (args->workspace_bytes < ws.total)
        return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "packed prefill workspace holds " + std::to_string(args->workspace_bytes) +
                                                         " bytes but the call needs " + std::to_string(ws.total));
    const uint64_t bytes = plane_bytes(args->num_blocks, PVLC_HIP_KV_F16);
    if (pvlc_hip_status st = apart({{args->key_cache, bytes}, {args->value_cache, bytes}, {args->workspace, ws.total}, outs},
                                   {queries, keys, values,
                                    {args->row_offsets, 4ull * args->num_seqs + 4},
                                    {args->block_tables, 4ull * args->num_seqs * args->max_blocks_per_seq},
                                    {args->cache_lens, 4ull * args->num_seqs},
                                    {args->positions, 4ull * args->rows},
                                    {args->rope_cos, 256ull * args->rope_rows},
                                    {args->rope_sin, 256ull * args->rope_rows}},
                                   "a packed prefill's planes, workspace and output"))
        return st;
    auto *base = static_cast<unsigned char *>(args->workspace);
    AppendRows a{};
    a.ragged = ragged_rows(args);
    a.code = PVLC_HIP_KV_F16;
    a.f32 = f32;
    a.key = key;
    a.value = value;
    a.key_stride = static_cast<int64_t>(key_stride);
    a.value_stride = static_cast<int64_t>(value_stride);
    a.rope_cos = args->rope_cos;
    a.rope_sin = args->rope_sin;
    a.rope_rows = args->rope_rows;
    a.positions = args->positions;
    a.key_cache = args->key_cache;
    a.value_cache = args->value_cache;
    a.error_word = reinterpret_cast<uint32_t *>(base);
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
    if (const int e = launch_kv_append(a, stream)) return hip_status(e, "packed prefill append launch");
    if (const int e = launch_packed_prefill(r, stream)) return hip_status(e, "packed prefill launch");
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
    return packed_workspace_layout(num_seqs, rows, max_context).total;
}

pvlc_hip_status pvlc_hip_packed_prefill_f16(const pvlc_hip_packed_prefill_args *args, const uint16_t *query, const uint16_t *key,
                                            const uint16_t *value, uint16_t *out, void *stream) {
    return prefill(args, query, key, value, out, false, stream);
}

pvlc_hip_status pvlc_hip_packed_prefill_f32io(const pvlc_hip_packed_prefill_args *args, const float *query, const float *key,
                                              const float *value, float *out, void *stream) {
    return prefill(args, query, key, value, out, true, stream);
}

}  // extern "C"
