// Entry points of serving over an 8-bit paged cache: argument checks before any
// GPU effect, then the launches.

#include <cstdint>
#include <string>

#include "pvlc_internal.hpp"

using namespace pvlc;

namespace {

// Workgroups of 256 threads that a launch may have (below 2^32 threads).
constexpr uint64_t kMaxGroups = 1u << 24;

bool aligned(const void *p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

pvlc_hip_status check_codes(uint32_t code, const void *keys, const void *values, const void *exponents) {
    if (code != PVLC_HIP_KV_E4M3 && code != PVLC_HIP_KV_INT8)
        return invalid(PVLC_HIP_INV_INVALID_ACTIVATION_LAYOUT, "the cache's code is PVLC_HIP_KV_E4M3 or PVLC_HIP_KV_INT8, not " + std::to_string(code));
    if (!keys || !values || !exponents) return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "8-bit cache plane or exponents pointer is NULL");
    if (!aligned(keys, 16) || !aligned(values, 16) || !aligned(exponents, 4))
        return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "8-bit cache planes must be 16-byte aligned, their exponents 4-byte aligned");
    return PVLC_HIP_OK;
}

pvlc_hip_status decode_q8(const pvlc_hip_paged_decode_q8_args *args, const DecodeOperands32 *f32, void *stream) {
    if (!args) return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "paged decode args are NULL");
    if (pvlc_hip_status st = check_codes(args->code, args->key_cache, args->value_cache, args->exponents)) return st;
    // The fp16 decode's arguments, checks and plan; its kernels alone differ.
    pvlc_hip_paged_decode_args a{};
    a.num_seqs = args->num_seqs;
    a.num_blocks = args->num_blocks;
    a.max_blocks_per_seq = args->max_blocks_per_seq;
    a.block_tables = args->block_tables;
    a.cache_lens = args->cache_lens;
    a.uniform_cache_len = args->uniform_cache_len;
    a.max_context = args->max_context;
    a.key_cache = reinterpret_cast<uint16_t *>(args->key_cache);
    a.value_cache = reinterpret_cast<uint16_t *>(args->value_cache);
    a.query = args->query;
    a.new_key = args->new_key;
    a.new_value = args->new_value;
    a.out = args->out;
    a.rope_cos = args->rope_cos;
    a.rope_sin = args->rope_sin;
    a.rope_rows = args->rope_rows;
    a.positions = args->positions;
    a.rotate_query = args->rotate_query;
    a.partition_tokens = args->partition_tokens;
    a.workspace = args->workspace;
    a.workspace_bytes = args->workspace_bytes;
    const DecodeCodes codes{args->code, args->exponents};
    if (pvlc_hip_status st = launch_decode_checked(&a, stream, nullptr, f32, &codes)) return st;
    return ok();
}

pvlc_hip_status check_rows(const void *keys, const void *values, uint64_t end, uint32_t tokens, const int32_t *table, uint32_t num_blocks) {
    if (!keys || !values) return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "row pointer is NULL");
    if (!aligned(keys, 2) || !aligned(values, 2)) return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "fp16 rows must be 2-byte aligned");
    if (tokens == 0 || num_blocks == 0) return invalid(PVLC_HIP_INV_ZERO_DIMENSION, "tokens and blocks must be nonzero");
    if (end > 0xFFFFFFF0ull) return invalid(PVLC_HIP_INV_ARITHMETIC_OVERFLOW, "the last token exceeds 32 bits");
    if (end / kBlockTokens >= kMaxGroups - 1) return invalid(PVLC_HIP_INV_INVALID_DECODER_GEOMETRY, "the blocks of a move exceed the grid");
    if (!table && (end + kBlockTokens - 1) / kBlockTokens > num_blocks)
        return invalid(PVLC_HIP_INV_INVALID_DECODER_GEOMETRY, "tokens exceed the contiguous blocks");
    return PVLC_HIP_OK;
}

// The pool's description checked, its planes and workspace laid out.
pvlc_hip_status check_pool(const pvlc_hip_kv_pool *pool, uint32_t rows, PagePlanes *planes, PagesWorkspace *layout) {
    if (!pool) return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "page pool is NULL");
    if (pool->num_blocks == 0 || pool->max_blocks_per_seq == 0 || pool->num_planes == 0 || pool->num_layers == 0)
        return invalid(PVLC_HIP_INV_ZERO_DIMENSION, "blocks, table width, planes and layers of a page pool must be nonzero");
    if (pool->num_blocks > 0x7FFFFFFFu || pool->num_planes > kMaxPagePlanes || pool->num_layers > 65535u)
        return invalid(PVLC_HIP_INV_INVALID_DECODER_GEOMETRY, "a page pool holds below 2^31 blocks, at most 4 planes and 65535 layers");
    if (rows > 65535u || static_cast<uint64_t>(rows) * pool->max_blocks_per_seq > 0x7FFFFFFFull)
        return invalid(PVLC_HIP_INV_INVALID_DECODER_GEOMETRY, "at most 65535 table rows and 2^31 - 1 entries");
    if (pool->max_blocks_per_seq > 0x7FFFFFFFu / kBlockTokens)
        return invalid(PVLC_HIP_INV_INVALID_DECODER_GEOMETRY, "a table row's tokens exceed 2^31 - 1");
    if (!pool->ref_counts || !pool->free_mask || !pool->workspace)
        return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "page pool counts, mask or workspace pointer is NULL");
    if (!aligned(pool->ref_counts, 4) || !aligned(pool->free_mask, 4) || !aligned(pool->workspace, 256))
        return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "page pool counts and mask must be 4-byte aligned, the workspace 256-byte aligned");
    *planes = {};
    planes->count = pool->num_planes;
    planes->layers = pool->num_layers;
    for (uint32_t i = 0; i < pool->num_planes; ++i) {
        const pvlc_hip_kv_plane &p = pool->planes[i];
        if (!p.base) return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "page plane " + std::to_string(i) + " is NULL");
        if (p.block_bytes == 0 || p.block_bytes % 4 != 0 || !aligned(p.base, 4) || p.layer_stride_bytes % 4 != 0)
            return invalid(PVLC_HIP_INV_INVALID_ACTIVATION_LAYOUT,
                           "page plane " + std::to_string(i) + " must be 4-byte aligned, with blocks and layers of a multiple of 4 bytes");
        if (p.block_bytes > 0x7FFFFFFFull) return invalid(PVLC_HIP_INV_ARITHMETIC_OVERFLOW, "a page's part of a plane exceeds 2^31 - 1 bytes");
        if (pool->num_layers > 1 && p.layer_stride_bytes < p.block_bytes * pool->num_blocks)
            return invalid(PVLC_HIP_INV_INVALID_ACTIVATION_LAYOUT, "layers of page plane " + std::to_string(i) + " overlap");
        if (p.layer_stride_bytes > UINT64_MAX / 65536u) return invalid(PVLC_HIP_INV_ARITHMETIC_OVERFLOW, "the layers of a page plane exceed 64 bits");
        const bool wide = aligned(p.base, 16) && p.block_bytes % 16 == 0 && p.layer_stride_bytes % 16 == 0;
        planes->plane[i] = {static_cast<uint8_t *>(p.base), nullptr, p.block_bytes, p.layer_stride_bytes, wide, 0};
    }
    *layout = pages_workspace_layout(pool->num_blocks, rows);
    if (pool->workspace_bytes < layout->total)
        return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "page workspace holds " + std::to_string(pool->workspace_bytes) +
                                                         " bytes but the call needs " + std::to_string(layout->total));
    return PVLC_HIP_OK;
}

bool overlap(const void *a, uint64_t a_bytes, const void *b, uint64_t b_bytes) {
    const auto x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a_bytes && b_bytes && x < y + b_bytes && y < x + a_bytes;
}

}  // namespace

extern "C" {

pvlc_hip_status pvlc_hip_paged_decode_q8_f16(const pvlc_hip_paged_decode_q8_args *args, void *stream) {
    return decode_q8(args, nullptr, stream);
}

pvlc_hip_status pvlc_hip_paged_decode_q8_f32io(const pvlc_hip_paged_decode_q8_args *args, const float *query, const float *new_key,
                                               const float *new_value, float *out, void *stream) {
    const DecodeOperands32 f32{query, new_key, new_value, out};
    return decode_q8(args, &f32, stream);
}

pvlc_hip_status pvlc_hip_kv_pack_q8(const uint16_t *key_rows, const uint16_t *value_rows, uint32_t first_token, uint32_t tokens,
                                    const int32_t *block_table, uint32_t num_blocks, uint32_t code, uint8_t *key_cache,
                                    uint8_t *value_cache, uint8_t *exponents, void *stream) {
    if (pvlc_hip_status st = check_codes(code, key_cache, value_cache, exponents)) return st;
    if (pvlc_hip_status st = check_rows(key_rows, value_rows, static_cast<uint64_t>(first_token) + tokens, tokens, block_table, num_blocks))
        return st;
    const int e = launch_kv_pack_q8(key_rows, value_rows, first_token, tokens, block_table, num_blocks, code, key_cache, value_cache,
                                    exponents, stream);
    if (e != 0) return hip_status(e, "8-bit kv pack launch");
    return ok();
}

pvlc_hip_status pvlc_hip_kv_unpack_q8(const uint8_t *key_cache, const uint8_t *value_cache, const uint8_t *exponents, uint32_t tokens,
                                      const int32_t *block_table, uint32_t num_blocks, uint32_t code, uint16_t *key_rows,
                                      uint16_t *value_rows, void *stream) {
    if (pvlc_hip_status st = check_codes(code, key_cache, value_cache, exponents)) return st;
    if (pvlc_hip_status st = check_rows(key_rows, value_rows, tokens, tokens, block_table, num_blocks)) return st;
    const int e = launch_kv_unpack_q8(key_cache, value_cache, exponents, tokens, block_table, num_blocks, code, key_rows, value_rows, stream);
    if (e != 0) return hip_status(e, "8-bit kv unpack launch");
    return ok();
}

size_t pvlc_hip_kv_pages_workspace_bytes(uint32_t num_blocks, uint32_t rows) {
    return num_blocks == 0 ? 0 : pages_workspace_layout(num_blocks, rows).total;
}

pvlc_hip_status pvlc_hip_kv_pages_reset(const pvlc_hip_kv_pool *pool, void *stream) {
    PagePlanes planes;
    PagesWorkspace ws;
    if (pvlc_hip_status st = check_pool(pool, 0, &planes, &ws)) return st;
    const int e = launch_pages_reset(pool->ref_counts, pool->free_mask, pool->num_blocks, static_cast<uint32_t *>(pool->workspace), stream);
    if (e != 0) return hip_status(e, "page pool reset launch");
    return ok();
}

pvlc_hip_status pvlc_hip_kv_pages_fork(const pvlc_hip_kv_pool *pool, const pvlc_hip_kv_fork_args *args, void *stream) {
    if (!args) return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "fork args are NULL");
    const uint32_t rows = args->rows_in > args->rows_out ? args->rows_in : args->rows_out;
    PagePlanes planes;
    PagesWorkspace ws;
    if (pvlc_hip_status st = check_pool(pool, rows, &planes, &ws)) return st;
    if (rows == 0) return invalid(PVLC_HIP_INV_ZERO_DIMENSION, "a fork needs input or output rows");
    if (rows > kMaxForkRows) return invalid(PVLC_HIP_INV_INVALID_DECODER_GEOMETRY, "a fork takes at most 4096 rows");
    if (args->rows_in && (!args->tables_in || !args->lens_in)) return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "fork input pointer is NULL");
    if (args->rows_out && (!args->tables_out || !args->lens_out)) return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "fork output pointer is NULL");
    for (const void *p : {static_cast<const void *>(args->tables_in), static_cast<const void *>(args->lens_in), static_cast<const void *>(args->parents),
                          static_cast<const void *>(args->reserve), static_cast<const void *>(args->tables_out), static_cast<const void *>(args->lens_out)})
        if (!aligned(p, 4)) return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "fork tables, lengths, parents and reserve must be 4-byte aligned");
    // A workgroup of 256 threads for each row and for each (row, layer).
    if (static_cast<uint64_t>(args->rows_out) * pool->num_layers + args->rows_in + args->rows_out >= kMaxGroups)
        return invalid(PVLC_HIP_INV_INVALID_DECODER_GEOMETRY, "rows times layers of a fork exceed the grid");
    const uint64_t width = static_cast<uint64_t>(pool->max_blocks_per_seq) * 4;
    const struct {
        const void *at;
        uint64_t bytes;
    } in[] = {{args->tables_in, args->rows_in * width},
              {args->lens_in, args->rows_in * 4ull},
              {args->parents, args->parents ? args->rows_out * 4ull : 0},
              {args->reserve, args->reserve ? args->rows_out * 4ull : 0}};
    for (const auto &i : in)
        if (overlap(i.at, i.bytes, args->tables_out, args->rows_out * width) || overlap(i.at, i.bytes, args->lens_out, args->rows_out * 4ull))
            return invalid(PVLC_HIP_INV_INVALID_ACTIVATION_LAYOUT, "a fork's output tables and lengths may not overlap its inputs");
    if (overlap(args->tables_out, args->rows_out * width, args->lens_out, args->rows_out * 4ull))
        return invalid(PVLC_HIP_INV_INVALID_ACTIVATION_LAYOUT, "a fork's output tables and lengths may not overlap");
    auto *base = static_cast<unsigned char *>(pool->workspace);
    PagesFork f{};
    f.num_blocks = pool->num_blocks;
    f.max_blocks = pool->max_blocks_per_seq;
    f.rows_in = args->rows_in;
    f.rows_out = args->rows_out;
    f.appended = args->appended;
    f.reserve_tokens = args->reserve_tokens;
    f.keep_inputs = args->keep_inputs != 0;
    f.tables_in = args->tables_in;
    f.lens_in = args->lens_in;
    f.parents = args->parents;
    f.reserve = args->reserve;
    f.tables_out = args->tables_out;
    f.lens_out = args->lens_out;
    f.ref_counts = pool->ref_counts;
    f.free_mask = pool->free_mask;
    f.plan = {reinterpret_cast<ForkRow *>(base + ws.rows_offset), reinterpret_cast<ForkInput *>(base + ws.inputs_offset),
              reinterpret_cast<int32_t *>(base + ws.first_offset), reinterpret_cast<uint32_t *>(base) + 1, reinterpret_cast<uint32_t *>(base)};
    const int e = launch_pages_fork(f, planes, stream);
    if (e != 0) return hip_status(e, "page fork launch");
    return ok();
}

pvlc_hip_status pvlc_hip_kv_pages_compact(const pvlc_hip_kv_pool *pool, int32_t *tables, uint32_t rows, int32_t *forward, void *stream) {
    PagePlanes planes;
    PagesWorkspace ws;
    if (pvlc_hip_status st = check_pool(pool, rows, &planes, &ws)) return st;
    if (rows && !tables) return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "compaction tables pointer is NULL");
    if (!aligned(tables, 4) || !aligned(forward, 4)) return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "compaction tables and map must be 4-byte aligned");
    if (overlap(tables, static_cast<uint64_t>(rows) * pool->max_blocks_per_seq * 4, forward, forward ? pool->num_blocks * 4ull : 0))
        return invalid(PVLC_HIP_INV_INVALID_ACTIVATION_LAYOUT, "a compaction's map may not overlap its tables");
    auto *base = static_cast<unsigned char *>(pool->workspace);
    PagesCompact c{};
    c.num_blocks = pool->num_blocks;
    c.max_blocks = pool->max_blocks_per_seq;
    c.rows = rows;
    c.tables = tables;
    c.forward = forward;
    c.ref_counts = pool->ref_counts;
    c.free_mask = pool->free_mask;
    c.plan = {reinterpret_cast<uint32_t *>(base + ws.words_offset), reinterpret_cast<int32_t *>(base + ws.first_offset),
              reinterpret_cast<int32_t *>(base + ws.second_offset), reinterpret_cast<int32_t *>(base + ws.third_offset),
              reinterpret_cast<uint32_t *>(base) + 2};
    const int e = launch_pages_compact(c, planes, stream);
    if (e != 0) return hip_status(e, "page compaction launch");
    return ok();
}

pvlc_hip_status pvlc_hip_kv_pages_copy(const pvlc_hip_kv_pool *from, const int32_t *from_blocks, const pvlc_hip_kv_pool *to, const int32_t *to_blocks,
                                       uint32_t count, void *stream) {
    PagePlanes source, planes;
    PagesWorkspace ws;
    if (pvlc_hip_status st = check_pool(from, 0, &source, &ws)) return st;
    if (pvlc_hip_status st = check_pool(to, 0, &planes, &ws)) return st;
    if (count == 0) return invalid(PVLC_HIP_INV_ZERO_DIMENSION, "a copy of pages needs pairs");
    if (count >= kMaxGroups) return invalid(PVLC_HIP_INV_INVALID_DECODER_GEOMETRY, "a copy of pages takes below 2^24 pairs");
    if (!from_blocks || !to_blocks || !aligned(from_blocks, 4) || !aligned(to_blocks, 4))
        return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "page lists must be given and 4-byte aligned");
    if (source.count != planes.count || source.layers != planes.layers)
        return invalid(PVLC_HIP_INV_INVALID_ACTIVATION_LAYOUT, "both pools of a copy need the same planes and layers");
    for (uint32_t i = 0; i < planes.count; ++i) {
        if (source.plane[i].block_bytes != planes.plane[i].block_bytes)
            return invalid(PVLC_HIP_INV_INVALID_ACTIVATION_LAYOUT, "plane " + std::to_string(i) + " has blocks of another size in the other pool");
        planes.plane[i].from = source.plane[i].base;
        planes.plane[i].from_stride = source.plane[i].layer_stride;
        planes.plane[i].wide = planes.plane[i].wide && source.plane[i].wide;
    }
    const int e = launch_pages_copy(from_blocks, to_blocks, count, from->num_blocks, to->num_blocks, planes, static_cast<uint32_t *>(to->workspace), stream);
    if (e != 0) return hip_status(e, "page copy launch");
    return ok();
}

size_t pvlc_hip_beam_workspace_bytes(uint32_t batch, uint32_t beams, uint32_t vocab, uint32_t best) {
    return batch == 0 || beams == 0 || vocab == 0 || best == 0 ? 0 : beam_workspace_layout(batch, beams, vocab, best).total;
}

pvlc_hip_status pvlc_hip_beam_select_f32(const pvlc_hip_beam_args *args, void *stream) {
    if (!args) return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "beam args are NULL");
    if (args->batch == 0 || args->beams == 0 || args->vocab == 0 || args->best == 0)
        return invalid(PVLC_HIP_INV_ZERO_DIMENSION, "batch, beams, vocab and best must be nonzero");
    if (args->beams > kBeamMaxBeams || args->best > kBeamMaxBest)
        return invalid(PVLC_HIP_INV_INVALID_DECODER_GEOMETRY, "at most 64 beams and 128 candidates");
    if (args->vocab > 0x7FFFFFFFu || static_cast<uint64_t>(args->batch) * args->beams > 65535u)
        return invalid(PVLC_HIP_INV_INVALID_DECODER_GEOMETRY, "below 2^31 logits a row and at most 65535 rows");
    const uint64_t rows = static_cast<uint64_t>(args->batch) * args->beams;
    const uint32_t segments = (args->vocab - 1) / kBeamSegment + 1;
    if (segments * rows >= kMaxGroups)
        return invalid(PVLC_HIP_INV_INVALID_DECODER_GEOMETRY, "rows times vocab of a beam selection exceed the grid");
    if (args->row_stride < args->vocab) return invalid(PVLC_HIP_INV_INVALID_ACTIVATION_LAYOUT, "rows of logits overlap");
    if (!args->logits || !args->scores || !args->next_scores || !args->parents || !args->tokens || !args->workspace)
        return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "beam buffer pointer is NULL");
    for (const void *p : {static_cast<const void *>(args->logits), static_cast<const void *>(args->scores), static_cast<const void *>(args->finished),
                          static_cast<const void *>(args->next_scores), static_cast<const void *>(args->parents), static_cast<const void *>(args->tokens),
                          static_cast<const void *>(args->next_finished)})
        if (!aligned(p, 4)) return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "beam buffers must be 4-byte aligned");
    if (args->row_stride > UINT64_MAX / 8 / rows) return invalid(PVLC_HIP_INV_ARITHMETIC_OVERFLOW, "the rows of logits exceed 64 bits");
    const uint64_t in = rows * 4, out = static_cast<uint64_t>(args->batch) * args->best * 4, read = ((rows - 1) * args->row_stride + args->vocab) * 4;
    const void *outputs[] = {args->next_scores, args->parents, args->tokens, args->next_finished};
    for (const void *p : outputs)
        if (overlap(p, p ? out : 0, args->scores, in) || overlap(p, p ? out : 0, args->finished, args->finished ? in : 0) ||
            overlap(p, p ? out : 0, args->logits, read))
            return invalid(PVLC_HIP_INV_INVALID_ACTIVATION_LAYOUT, "the selection's outputs may not overlap its logits, scores or finished flags");
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < i; ++j)
            if (overlap(outputs[i], outputs[i] ? out : 0, outputs[j], outputs[j] ? out : 0))
                return invalid(PVLC_HIP_INV_INVALID_ACTIVATION_LAYOUT, "the selection's outputs may not overlap one another");
    const BeamWorkspace ws = beam_workspace_layout(args->batch, args->beams, args->vocab, args->best);
    if (args->workspace_bytes < ws.total)
        return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "beam workspace holds " + std::to_string(args->workspace_bytes) + " bytes but the call needs " +
                                                         std::to_string(ws.total));
    if (!aligned(args->workspace, 256)) return invalid(PVLC_HIP_INV_LENGTH_MISMATCH, "beam workspace must be 256-byte aligned");
    auto *base = static_cast<unsigned char *>(args->workspace);
    BeamSelect b{};
    b.batch = args->batch;
    b.beams = args->beams;
    b.vocab = args->vocab;
    b.best = args->best;
    b.segments = segments;
    b.row_stride = args->row_stride;
    b.logits = args->logits;
    b.scores = args->scores;
    b.finished = args->finished;
    b.end_token = args->end_token;
    b.next_scores = args->next_scores;
    b.parents = args->parents;
    b.tokens = args->tokens;
    b.next_finished = args->next_finished;
    b.arrived = reinterpret_cast<uint32_t *>(base);
    b.keys = reinterpret_cast<uint64_t *>(base + ws.keys_offset);
    b.sums = reinterpret_cast<double *>(base + ws.sums_offset);
    b.references = reinterpret_cast<float *>(base + ws.references_offset);
    b.row_keys = reinterpret_cast<uint64_t *>(base + ws.row_keys_offset);
    b.row_tokens = reinterpret_cast<uint64_t *>(base + ws.row_tokens_offset);
    const int e = launch_beam_select(b, stream);
    if (e != 0) return hip_status(e, "beam selection launch");
    return ok();
}

}  // extern "C"
