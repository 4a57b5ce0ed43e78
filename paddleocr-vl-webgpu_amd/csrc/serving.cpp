// Entry points of serving over an 8-bit paged cache: argument checks before any
// GPU effect, then the launches.

#include <cstdint>
#include <string>

#include "pvlc_internal.hpp"

using namespace pvlc;

namespace {

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
    if (!table && (end + kBlockTokens - 1) / kBlockTokens > num_blocks)
        return invalid(PVLC_HIP_INV_INVALID_DECODER_GEOMETRY, "tokens exceed the contiguous blocks");
    return PVLC_HIP_OK;
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

}  // extern "C"
