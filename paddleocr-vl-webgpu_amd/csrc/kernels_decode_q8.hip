// Paged GQA decode over an 8-bit cache for gfx950: fused rotary, append and
// split-K attention.
//
// Per kv head, with codes kc, vc and the exponents ek, ev of their block
// (pvlc_q8.hpp), and s_t = log2(e) / sqrt(128) 2^ek (q . kc_t) in log2 units:
//   o = sum_t 2^s_t 2^ev vc_t / sum_t 2^s_t.
// One running reference M = max_t (s_t + ev) serves both sums: the weights
// 2^(s_t - M) 2^ev that multiply the codes are at most 1, and the terms
// 2^(s_t - M) of the denominator at most 2^-ev <= 2^32.
//
// The codes become fp16 in registers for the scores (v_mfma_f32_16x16x32_f16) and
// bf16 for P.V (v_mfma_f32_16x16x32_bf16), both exactly.  A wave takes 64 tokens
// (four blocks) of one head at a time, all in 16-byte loads:
//   keys    load (h, half): lane (row, kg) the dims half*64 + kg*16 .. +16 of
//           token h*4 + row%4 of tile row/4; its low and high eight codes are
//           the operands of two score MFMAs, and score MFMA chain h leaves lane
//           (head, kg) the tokens h*4 .. h*4+3 of tile kg;
//   values  load cc: lane (row, kg) all 16 tokens of dim cc*16 + row of tile kg;
//           the low and high eight are the operands of two P.V MFMAs, whose
//           weights the lane (head, kg) holds.
// The key slab [token/4][dim/16][token%4][dim%16] makes each load of a tile 256
// contiguous bytes; the value slab [dim][token] does as it is.
//
// The weights go to P.V as sums of bf16 terms, three for f32 operands (all 24
// bits) and two for fp16 ones (16 bits, so that the output is rounded once: with one fp16
// term it was off by two roundings).  bf16 has the exponents of f32, which a weight
// needs: a block whose values are 2^k times larger than another's pushes that one's
// weights 2^k below the reference, up to 2^40, while in the dims where it is not
// larger they count as much as its own.  (fp16 terms lost them: with one value of
// 30000 among others of 1 those dims were off by 6e-4, of 0.05 by 1.3e-2.)  The third
// term costs 0.2 us of a launch's 8 with f32 operands, the pair 0.2-0.4 of a single
// one's 7.2-9.1 with fp16 ones.
//
// What bounds it.  512 bytes a token and 8192 operations: memory, once a launch is
// long.  256 sequences of 1024 to 32768 rows (1.20 GB): 216-222 us (int8 221-232,
// with f32 operands 223-244) and the merge 8-9, 5.4 TB/s, where a copy reaches 5.1;
// the fp16 cache's takes 453 us.  Short launches are a chain of rounds: one
// sequence of 1157 rows 7.8 us (f32 operands), thirteen up to 2010 7.9, 18 caches
// of 2048 rows (19 MB) 9.5 in e4m3 and 10.0 in int8, whose conversion takes more
// instructions; in int8 with f32 operands 8.2, 8.9 and 10.7.  Time stamps of the
// waves put 0.75 us of that into the new row (its rounding and the LDS detour to
// the wave's own registers), 0.8 into the hand-off and 1.3 into the merge; the
// rest is the launch, the block ids and one round of loads.  Measured slower and
// not kept: the merge's loads issued for every slot without a branch, and the new
// row's codes read from LDS ahead of the loop.

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "decode_device.hpp"
#include "pvlc_q8.hpp"

namespace pvlc {
namespace {

struct DecodeQ8Params : DecodeParams {
    uint8_t *exponents;  // [block][kv head][key, value], biased by 127
};

constexpr int kTiles = 4;                  // 16-token tiles of a wave's chunk
constexpr int kChunkTokens = kTiles * 16;

// Combine the waves of a partition in LDS, then write the output, store the
// partial (DEFER_MERGE, for paged_decode_merge_kernel) or, as the last
// partition to arrive, merge them all.  m_run and l_run belong to head
// lane % 16, o[c][r] to head (lane / 16) * 4 + r at dim c * 16 + lane % 16.
// The hand-off is decode_device.hpp's.
template <int WAVES, bool DEFER_MERGE, bool F32IO>
__device__ inline void finish_item(const DecodeParams &p, uint32_t s, uint32_t g, uint32_t part, int num_parts,
                                   float m_run, float l_run, const float4_t (&o)[8]) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int row = lane & 15, kg = lane >> 4;
    __shared__ float sm_m[WAVES][kGroup];
    __shared__ float sm_l[WAVES][kGroup];
    __shared__ __align__(16) float sm_o[WAVES][kGroup][kHeadDim + 4];
    __shared__ int sm_last;
    if (lane < static_cast<int>(kGroup)) {
        sm_m[wave][lane] = m_run;
        sm_l[wave][lane] = l_run;
    }
    if (kg < 2) {
#pragma unroll
        for (int c = 0; c < 8; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) sm_o[wave][kg * 4 + r][c * 16 + row] = o[c][r];
    }
    __syncthreads();

    // Each of the first kCT threads owns kPer (a multiple of 4) consecutive
    // elements of one head; the others shadow thread 0 and store nothing.
    constexpr int kCT = WAVES >= 4 ? 256 : (WAVES >= 2 ? 128 : 64);
    constexpr int kPer = (kGroup * kHeadDim) / kCT;
    static_assert(kPer % 4 == 0, "16-byte pieces");
    const bool active = threadIdx.x < kCT;
    const int e0 = active ? static_cast<int>(threadIdx.x) * kPer : 0;
    const int h = e0 >> 7, d0 = e0 & 127;
    float mw[WAVES], lw[WAVES];
    float4_t ow[WAVES][kPer / 4];
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        mw[w] = sm_m[w][h];
        lw[w] = sm_l[w][h];
#pragma unroll
        for (int e = 0; e < kPer / 4; ++e) ow[w][e] = *reinterpret_cast<const float4_t *>(&sm_o[w][h][d0 + e * 4]);
    }
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) M = fmaxf(M, mw[w]);
    float L = 0.f;
    float4_t po[kPer / 4] = {};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const float f = __builtin_amdgcn_exp2f(mw[w] - M);  // 0 for a wave without tokens
        L += lw[w] * f;
#pragma unroll
        for (int e = 0; e < kPer / 4; ++e) po[e] += ow[w][e] * f;
    }
    const size_t out_off = (static_cast<size_t>(s) * kQueryHeads + g * kGroup) * kHeadDim + e0;
    auto put = [&](const float4_t (&v)[kPer / 4], float inv) {
        if (!active) return;
#pragma unroll
        for (int e = 0; e < kPer / 4; ++e) {
            const float4_t r = v[e] * inv;
            if constexpr (F32IO) {
                *reinterpret_cast<float4_t *>(p.out32 + out_off + e * 4) = r;
            } else {
                const half4_t q = {to_h(r[0]), to_h(r[1]), to_h(r[2]), to_h(r[3])};
                *reinterpret_cast<half4_t *>(p.out + out_off + e * 4) = q;
            }
        }
    };
    if (num_parts == 1) return put(po, 1.0f / L);

    const size_t unit = (static_cast<size_t>(s) * kKvHeads + g) * p.part_stride;
    float *part_o = p.part_o + (unit + part) * (kGroup * kHeadDim);
    float *part_ml = p.part_ml + (unit + part) * (2 * kGroup);  // [head][max, sum]
    if constexpr (DEFER_MERGE) {
        if (active) {
#pragma unroll
            for (int e = 0; e < kPer / 4; ++e) *reinterpret_cast<float4_t *>(part_o + e0 + e * 4) = po[e];
            if (d0 == 0) {
                part_ml[2 * h] = M;
                part_ml[2 * h + 1] = L;
            }
        }
        return;
    } else {
        const __amdgpu_buffer_rsrc_t rsrc = partials_buffer(p, unit);
        if (active) {
#pragma unroll
            for (int e = 0; e < kPer / 4; ++e) store_partial_sc1(rsrc, part * (kGroup * kHeadDim) + e0 + e * 4, __builtin_bit_cast(u32x4_t, po[e]));
            if (d0 == 0) store_pair_sc1(part_ml + 2 * h, M, L);
        }
        if (!last_to_arrive(p, s, g, part, num_parts, sm_last)) return;

        const float *all_ml = p.part_ml + unit * (2 * kGroup);
        constexpr int kBatch = kPer >= 16 ? 4 : (kPer >= 8 ? 8 : 16);
        float Mg = -INFINITY, Lg = 0.f;
        float4_t og[kPer / 4] = {};
        for (int q0 = 0; q0 < num_parts; q0 += kBatch) {
            float mv[kBatch], lv[kBatch];
            float4_t ov[kBatch][kPer / 4];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const int q = q0 + b;
                mv[b] = M;
                lv[b] = L;
#pragma unroll
                for (int e = 0; e < kPer / 4; ++e) ov[b][e] = po[e];  // its own, or a stand-in past the last (weight 0)
                if (q < num_parts && q != static_cast<int>(part)) {  // uniform
                    load_pair_sc1(all_ml + q * (2 * kGroup) + 2 * h, &mv[b], &lv[b]);
#pragma unroll
                    for (int e = 0; e < kPer / 4; ++e)
                        ov[b][e] = __builtin_bit_cast(float4_t, load_partial_sc1(rsrc, q * (kGroup * kHeadDim) + e0 + e * 4));
                }
            }
            float Mb = Mg;
#pragma unroll
            for (int b = 0; b < kBatch; ++b)
                if (q0 + b < num_parts) Mb = fmaxf(Mb, mv[b]);
            const float a = __builtin_amdgcn_exp2f(Mg - Mb);
            Lg *= a;
#pragma unroll
            for (int e = 0; e < kPer / 4; ++e) og[e] *= a;
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const float w = (q0 + b < num_parts) ? __builtin_amdgcn_exp2f(mv[b] - Mb) : 0.f;
                Lg += lv[b] * w;
#pragma unroll
                for (int e = 0; e < kPer / 4; ++e) og[e] += ov[b][e] * w;
            }
            Mg = Mb;
        }
        put(og, 1.0f / Lg);
    }
}

// The keys and values of chunk c of this wave (block ids one per lane in ids).
// A tile's 16 bytes of a load lie 256 bytes behind those of the load before.
__device__ inline void load_chunk(const DecodeParams &p, uint32_t g, uint32_t ids, int c, int row, int kg,
                                  q8x4_t (&kr)[8], q8x4_t (&vr)[8]) {
    auto id = [&](int i) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(ids), c * kTiles + i)); };
    const uint32_t b0 = id(0), b1 = id(1), b2 = id(2), b3 = id(3);
    const uint32_t kb = (row & 8) ? ((row & 4) ? b3 : b2) : ((row & 4) ? b1 : b0);  // tile row / 4
    const uint32_t vb = (kg & 2) ? ((kg & 1) ? b3 : b2) : ((kg & 1) ? b1 : b0);
    const uint8_t *kp = reinterpret_cast<const uint8_t *>(p.key_cache) +
                        (static_cast<size_t>(kb) * kKvHeads + g) * kQ8SlabBytes + (kg * 4 + (row & 3)) * 16;
    const uint8_t *vp = reinterpret_cast<const uint8_t *>(p.value_cache) +
                        (static_cast<size_t>(vb) * kKvHeads + g) * kQ8SlabBytes + row * 16;
#pragma unroll
    for (int i = 0; i < 8; ++i) kr[i] = __builtin_nontemporal_load(reinterpret_cast<const q8x4_t *>(kp + i * 256));
    __builtin_amdgcn_sched_barrier(0);  // the keys ahead of the values
#pragma unroll
    for (int i = 0; i < 8; ++i) vr[i] = __builtin_nontemporal_load(reinterpret_cast<const q8x4_t *>(vp + i * 256));
}

// One work item: partition `part` (P tokens) of kv head g of sequence s, as
// decode_item of the fp16 cache.
template <int WAVES, bool DEFER_MERGE, bool F32IO, int CODE>
__device__ inline void decode_q8_item(const DecodeQ8Params &p, int P, uint32_t s, uint32_t g, uint32_t part, int cache_len,
                                      int pos, uint32_t ids, bool ids_bad) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int row = lane & 15, kg = lane >> 4;
    const int T = cache_len + 1;
    const int part_start = static_cast<int>(part) * P;
    if (part_start >= T) return;
    const int part_end = min(part_start + P, T);
    const int num_parts = (T + P - 1) / P;

    // Exponents of the wave's tiles, where their block ids are: key in the low
    // byte, value in the high one.
    uint32_t ex = *reinterpret_cast<const uint16_t *>(p.exponents + (static_cast<size_t>(ids) * kKvHeads + g) * 2);

    // Every pointer of the small operands in one round of scalar loads, and the
    // operands raw, on every lane and without a branch (cos and sin read the new
    // key row where there is no rotary): arithmetic between them and the cache's
    // loads would wait for them before those go out.
    asm volatile("" ::"s"(p.rope_cos), "s"(p.rope_sin), "s"(p.rope_rows));
    bool rope = p.rope_cos != nullptr;
    const bool rope_bad = rope && (pos < 0 || static_cast<uint32_t>(pos) >= p.rope_rows);
    if (rope_bad) rope = false;

    // The query, B operand of the score MFMAs: column = head of the group (8
    // real, 8 zero), step kb of a lane the dims (kb/2)*64 + kg*16 + (kb%2)*8
    // .. +8.  The new row: lane t has dims t and t + 64.
    const size_t qoff = (static_cast<size_t>(s) * kQueryHeads + g * kGroup + (row & 7)) * kHeadDim + kg * 16;
    const size_t new_base = (static_cast<size_t>(s) * kKvHeads + g) * kHeadDim;
    const float *stand_in = F32IO ? p.new_key32 + new_base : reinterpret_cast<const float *>(p.new_key + new_base);
    const float rc_raw = (rope ? p.rope_cos + static_cast<size_t>(pos) * 64 : stand_in)[lane];
    const float rs_raw = (rope ? p.rope_sin + static_cast<size_t>(pos) * 64 : stand_in)[lane];
    half8_t qb[4];
    float4_t q32[F32IO ? 4 : 1][2];
    float n32[4];  // key dims lane and lane + 64, value likewise
    uint16_t n16[4];
    if constexpr (F32IO) {
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
            const float *src = p.query32 + qoff + (kb >> 1) * 64 + (kb & 1) * 8;
            q32[kb][0] = *reinterpret_cast<const float4_t *>(src);
            q32[kb][1] = *reinterpret_cast<const float4_t *>(src + 4);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) n32[i] = (i < 2 ? p.new_key32 : p.new_value32)[new_base + lane + (i & 1) * 64];
    } else {
#pragma unroll
        for (int kb = 0; kb < 4; ++kb)
            qb[kb] = *reinterpret_cast<const half8_t *>(p.query + qoff + (kb >> 1) * 64 + (kb & 1) * 8);
#pragma unroll
        for (int i = 0; i < 4; ++i) n16[i] = (i < 2 ? p.new_key : p.new_value)[new_base + lane + (i & 1) * 64];
    }
    __builtin_amdgcn_sched_barrier(0);

    q8x4_t kr[8], vr[8];
    load_chunk(p, g, ids, 0, row, kg, kr, vr);
    __builtin_amdgcn_sched_barrier(0);

    if constexpr (!F32IO) {
#pragma unroll
        for (int i = 0; i < 4; ++i) n32[i] = static_cast<float>(__builtin_bit_cast(_Float16, n16[i]));
    }
    const float nk_lo = n32[0], nk_hi = n32[1], nv_lo = n32[2], nv_hi = n32[3];
    const float rc = rope ? rc_raw : 1.f, rs = rope ? rs_raw : 0.f;

    if (rope && p.rotate_query) {
        // The partner of step kb is step kb ^ 2 of the same lane; cos and sin
        // of pair i live in lane i.
        half8_t qr[4];
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int pair = kg * 16 + (kb & 1) * 8 + j;
                const float c = __shfl(rc, pair), sn = __shfl(rs, pair);
                float x, y;
                if constexpr (F32IO) {
                    x = q32[kb][j >> 2][j & 3];
                    y = q32[kb ^ 2][j >> 2][j & 3];
                } else {
                    x = static_cast<float>(qb[kb][j]);
                    y = static_cast<float>(qb[kb ^ 2][j]);
                }
                qr[kb][j] = kb < 2 ? to_h(x * c + (-y) * sn) : to_h(x * c + y * sn);
            }
        }
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) qb[kb] = qr[kb];
    } else if constexpr (F32IO) {
#pragma unroll
        for (int kb = 0; kb < 4; ++kb)
#pragma unroll
            for (int j = 0; j < 8; ++j) qb[kb][j] = to_h(q32[kb][j >> 2][j & 3]);
    }
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
        if (row >= static_cast<int>(kGroup)) qb[kb] = half8_t{};

    // Append: the wave whose tiles hold the new row's block rotates the row,
    // rounds it to fp16 as the fp16 cache would hold it, finds the block's
    // exponents with it, writes the row's codes and leaves them in LDS to stand
    // in for that row of its own loads.  Only that wave reads the block, so no
    // barrier is needed.  Where an exponent grows (seldom), the rows before are
    // rounded again in the cache first, and read again.
    const int append_tile = cache_len >> 4, slot = cache_len & 15;
    const int rel = append_tile - (part_start >> 4);
    const bool appends = rel >= 0 && append_tile * 16 < part_end && wave == (rel / kTiles) % WAVES;
    const int append_chunk = appends ? rel / (kTiles * WAVES) : -1;
    const int ti = rel & (kTiles - 1);
    __shared__ __align__(16) uint8_t sm_new[2][kHeadDim];
    if (appends) {
        float k_lo = nk_lo, k_hi = nk_hi;
        if (rope) {
            k_lo = nk_lo * rc + (-nk_hi) * rs;
            k_hi = nk_hi * rc + nk_lo * rs;
        }
        auto held = [](float x) { return q8_value(static_cast<float>(to_h(x))); };
        k_lo = held(k_lo);
        k_hi = held(k_hi);
        const float v_lo = held(nv_lo), v_hi = held(nv_hi);
        const int at = append_chunk * kTiles + ti;  // the lane of the block's id
        const uint32_t blk = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(ids), at));
        const uint32_t old = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(ex), at));
        const int old_k = static_cast<int>(old & 255) - kQ8Bias, old_v = static_cast<int>(old >> 8) - kQ8Bias;
        int e_k = q8_exponent<CODE>(wave_max(q8_size(q8_size(0.f, k_lo), k_hi)));
        int e_v = q8_exponent<CODE>(wave_max(q8_size(q8_size(0.f, v_lo), v_hi)));
        if (slot > 0) {
            e_k = max(e_k, old_k);
            e_v = max(e_v, old_v);
        }
        const float pk = exp2_whole(-e_k), pv = exp2_whole(-e_v);
        const uint32_t codes = q8_encode<CODE>(k_lo * pk, k_hi * pk, v_lo * pv, v_hi * pv);
        sm_new[0][lane] = static_cast<uint8_t>(codes);
        sm_new[0][lane + 64] = static_cast<uint8_t>(codes >> 8);
        sm_new[1][lane] = static_cast<uint8_t>(codes >> 16);
        sm_new[1][lane + 64] = static_cast<uint8_t>(codes >> 24);
        const uint32_t now = static_cast<uint32_t>(e_k + kQ8Bias) | static_cast<uint32_t>(e_v + kQ8Bias) << 8;
        if (lane == at) ex = now;
        if (!__builtin_amdgcn_readlane(static_cast<int>(ids_bad), at)) {  // (a bad id reads block 0 and writes nothing)
            const size_t slab = static_cast<size_t>(blk) * kKvHeads + g;
            uint8_t *ks = reinterpret_cast<uint8_t *>(p.key_cache) + slab * kQ8SlabBytes;
            uint8_t *vs = reinterpret_cast<uint8_t *>(p.value_cache) + slab * kQ8SlabBytes;
            const int grown = __builtin_amdgcn_readfirstlane(slot > 0 ? (e_k - old_k) | (e_v - old_v) << 16 : 0);
            if (grown != 0) {
                requantise_block<CODE>(ks, vs, lane, slot, grown & 0xFFFF, grown >> 16);
                if (append_chunk == 0) load_chunk(p, g, ids, 0, row, kg, kr, vr);
            }
            // key (slot, d) at (slot/4)*512 + (d/16)*64 + (slot%4)*16 + d%16, value at d*16 + slot
            uint8_t *kd = ks + (slot >> 2) * 512 + (slot & 3) * 16 + (lane >> 4) * 64 + (lane & 15), *vd = vs + lane * 16 + slot;
            kd[0] = static_cast<uint8_t>(codes);
            kd[256] = static_cast<uint8_t>(codes >> 8);
            vd[0] = static_cast<uint8_t>(codes >> 16);
            vd[1024] = static_cast<uint8_t>(codes >> 24);
            if (lane == 0) *reinterpret_cast<uint16_t *>(p.exponents + slab * 2) = static_cast<uint16_t>(now);
        }
    }

    float m_run = -INFINITY;  // running reference of head `row`
    float l_run = 0.f;        // this lane's share of the running sum
    float4_t o[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) o[c] = float4_t{0.f, 0.f, 0.f, 0.f};

    // One chunk.  The first is code of its own, with nothing to rescale: as a turn
    // of the loop it took one sequence of 1157 rows 8.5 us against 7.9.
    auto attend = [&](auto first, int chunk, int ws) {
        constexpr bool kFirst = decltype(first)::value;
        if (chunk == append_chunk) {  // uniform
            // The new row's codes into the block's registers; the codes behind it
            // become 0 (they may be e4m3 NaN).  All from LDS before any is used.
            q8x4_t piece[2];
            uint32_t code[8];
#pragma unroll
            for (int i = 0; i < 2; ++i) piece[i] = *reinterpret_cast<const q8x4_t *>(&sm_new[0][i * 64 + kg * 16]);
#pragma unroll
            for (int i = 0; i < 8; ++i) code[i] = sm_new[1][i * 16 + row];
            const bool key_lane = (row >> 2) == ti && (row & 3) == (slot & 3);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (key_lane && (i >> 1) == (slot >> 2)) kr[i] = piece[i & 1];
            const int shift = (slot & 3) * 8;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const uint32_t before = w < (slot >> 2) ? ~0u : (w == (slot >> 2) ? (1u << shift) - 1u : 0u);
                const uint32_t keep = kg == ti ? before : ~0u, put = kg == ti && w == (slot >> 2) ? 0xFFu << shift : 0u;
#pragma unroll
                for (int i = 0; i < 8; ++i) vr[i][w] = (vr[i][w] & keep) | ((code[i] << shift) & put);
            }
        }
        // Tiles past the end repeat the last one, whose codes behind the new row
        // may be NaN and whose exponents may never have been written.
        const bool past = ws + kg * 16 >= part_end;
        if (ws + kChunkTokens > part_end && past) {
#pragma unroll
            for (int i = 0; i < 8; ++i) vr[i] = q8x4_t{0, 0, 0, 0};
        }

        // Exponents of tile kg, and its scores.
        const uint32_t te = static_cast<uint32_t>(__shfl(static_cast<int>(ex), chunk * kTiles + kg));
        const int ek = static_cast<int>(te & 255) - kQ8Bias, ev = static_cast<int>(te >> 8) - kQ8Bias;
        const float sk = p.scale_log2 * exp2_whole(ek);
        float x[16];
        float cmax = -INFINITY;
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            float4_t acc = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kb = 0; kb < 4; ++kb) {
                const q8x4_t w = kr[h * 2 + (kb >> 1)];
                acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(q8_half8<CODE>(w[(kb & 1) * 2], w[(kb & 1) * 2 + 1]), qb[kb], acc, 0, 0, 0);
            }
            const int tbase = ws + kg * 16 + h * 4;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                x[h * 4 + r] = (tbase + r < part_end) ? acc[r] * sk : -INFINITY;
                cmax = fmaxf(cmax, x[h * 4 + r]);
            }
        }
        cmax += static_cast<float>(ev);
        cmax = fmaxf(cmax, __shfl_xor(cmax, 16));
        cmax = fmaxf(cmax, __shfl_xor(cmax, 32));
        const float m_new = fmaxf(m_run, cmax);
        if constexpr (!kFirst) {
            const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
            l_run *= alpha;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float a = __shfl(alpha, kg * 4 + r);
#pragma unroll
                for (int c = 0; c < 8; ++c) o[c][r] *= a;
            }
        }
        m_run = m_new;

        const float pv = past ? 0.f : exp2_whole(ev);
        // Eight tokens' terms at a time and, side by side, the products of four times
        // 16 dims.  In the widest workgroups, whose waves have 168 registers, the dims
        // follow one another in the schedule too: else the compiler converts all of them
        // first, and spills (18 caches of 4000 rows, int8 and f32 operands, 14.2 us
        // against 17.3; the others are 0.05-0.1 us faster as they are).
        constexpr int kTerms = F32IO ? 3 : 2, kSide = 4;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            q8x4_t terms[kTerms];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float2_t w;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float pf = __builtin_amdgcn_exp2f(x[u * 8 + i * 2 + j] - m_new);
                    l_run += pf;
                    w[j] = pf * pv;
                }
#pragma unroll
                for (int k = 0; k < kTerms; ++k) {
                    const uint32_t r = __builtin_bit_cast(uint32_t, __builtin_convertvector(w, bf16x2_t));
                    terms[k][i] = r;
                    w -= float2_t{__uint_as_float(r << 16), __uint_as_float(r & 0xFFFF0000u)};  // exact in f32
                }
            }
#pragma unroll
            for (int c0 = 0; c0 < 8; c0 += kSide) {
                if constexpr (WAVES > 8) __builtin_amdgcn_sched_barrier(0);
                bf16x8_t v[kSide];
#pragma unroll
                for (int c = 0; c < kSide; ++c) v[c] = q8_bf16x8<CODE>(vr[c0 + c][u * 2], vr[c0 + c][u * 2 + 1]);
#pragma unroll
                for (int k = 0; k < kTerms; ++k)
#pragma unroll
                    for (int c = 0; c < kSide; ++c)
                        o[c0 + c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, terms[k]), v[c], o[c0 + c], 0, 0, 0);
            }
        }
    };
    int ws = part_start + wave * kChunkTokens;
    if (ws < part_end) attend(std::true_type{}, 0, ws);
    for (int chunk = 1; (ws += WAVES * kChunkTokens) < part_end; ++chunk) {
        load_chunk(p, g, ids, chunk, row, kg, kr, vr);
        attend(std::false_type{}, chunk, ws);
    }
    l_run += __shfl_xor(l_run, 16);
    l_run += __shfl_xor(l_run, 32);
    // Errors, once the loads are consumed: 2 = a block id outside the planes,
    // 4 = a rotary position outside the tables.
    if (__any(ids_bad) && lane == 0) atomicOr(p.error_word, 2u);
    if (rope_bad && threadIdx.x == 0) atomicOr(p.error_word, 4u);
    finish_item<WAVES, DEFER_MERGE, F32IO>(p, s, g, part, num_parts, m_run, l_run, o);
}

// Grid (partition, kv head, sequence).
// What the first loads' addresses need comes ahead of the parameter block, as
// scalars: the first 14 dwords of arguments are in SGPRs when a wave starts.
template <int WAVES, bool F32IO, int CODE>
__global__ __launch_bounds__(WAVES * 64, 2) void paged_decode_q8_kernel(uint16_t *key_cache, uint16_t *value_cache, uint8_t *exponents,
                                                                        const int32_t *cache_lens, const int32_t *block_tables,
                                                                        uint32_t uniform_cache_len, uint32_t max_blocks_per_seq,
                                                                        uint32_t num_blocks, uint32_t partition_and_parts,
                                                                        DecodeQ8Params p) {
    p.key_cache = key_cache;
    p.value_cache = value_cache;
    p.exponents = exponents;
    p.cache_lens = cache_lens;
    p.block_tables = block_tables;
    p.uniform_cache_len = uniform_cache_len;
    p.max_blocks_per_seq = max_blocks_per_seq;
    p.num_blocks = num_blocks;
    p.partition_tokens = partition_and_parts & 0xffffu;
    p.max_parts = partition_and_parts >> 16;
    // The pointers of the small operands in the first round of scalar loads.
    asm volatile("" ::"s"(p.positions), "s"(p.rope_cos), "s"(p.rope_sin), "s"(p.rope_rows));
    if constexpr (F32IO) asm volatile("" ::"s"(p.query32), "s"(p.new_key32), "s"(p.new_value32));
    else asm volatile("" ::"s"(p.query), "s"(p.new_key), "s"(p.new_value));
    const uint32_t part = blockIdx.x, g = blockIdx.y, s = blockIdx.z;
    if ((part | g | s) == 0 && p.partition_word != nullptr && threadIdx.x == 0) {
        p.partition_word[0] = p.partition_tokens;
        p.partition_word[1] = kTargetWorkgroups;
    }
    const int64_t len = checked_cache_len(p, p.cache_lens ? load_const(p.cache_lens, s) : static_cast<int64_t>(p.uniform_cache_len));
    if (len < 0) {
        if (part == 0 && g == 0 && threadIdx.x == 0) atomicOr(p.error_word, 1u);
        return;
    }
    const int cache_len = static_cast<int>(len), P = static_cast<int>(p.partition_tokens);
    const int part_start = static_cast<int>(part) * P;
    if (part_start > cache_len) return;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    bool bad = false;
    const uint32_t ids = wave_tile_ids<WAVES, kTiles>(p, s, part_start, min(part_start + P, cache_len + 1), wave, &bad);
    const int pos = p.positions ? load_const(p.positions, s) : cache_len;
    decode_q8_item<WAVES, false, F32IO, CODE>(p, P, s, g, part, cache_len, pos, ids, bad);
}

// Ragged lengths and long contexts: the persistent walk over the items.
template <int WAVES, bool F32IO, int CODE>
__global__ __launch_bounds__(WAVES * 64, 2) void paged_decode_q8_ragged_kernel(DecodeQ8Params p, uint32_t num_seqs) {
    ragged_items<WAVES, kTiles>(p, num_seqs, [&](int P, uint32_t s, uint32_t g, uint32_t part, int len, int pos,
                                                 uint32_t ids, bool bad) {
        decode_q8_item<WAVES, true, F32IO, CODE>(p, P, s, g, part, len, pos, ids, bad);
    });
}

template <bool F32IO, int CODE>
int launch_kernels(const DecodeLaunch &launch, DecodeQ8Params &p, hipStream_t st) {
    const pvlc_hip_paged_decode_args &a = *launch.args;
    if (launch.streaming) {
        int e = 0;
        const uint64_t max_items = static_cast<uint64_t>(launch.max_parts) * kKvHeads * a.num_seqs;
        const uint32_t wgs = resident_workgroups(reinterpret_cast<const void *>(&paged_decode_q8_ragged_kernel<4, F32IO, CODE>), 256,
                                                 max_items, &p.compute_units, &e);
        if (e != 0) return e;
        hipLaunchKernelGGL((paged_decode_q8_ragged_kernel<4, F32IO, CODE>), dim3(wgs), dim3(256), 0, st, p, a.num_seqs);
        hipLaunchKernelGGL(paged_decode_merge_kernel<F32IO>, dim3(kKvHeads, a.num_seqs), dim3(256), 0, st, static_cast<DecodeParams>(p));
        return static_cast<int>(hipGetLastError());
    }
    const dim3 grid(launch.max_parts, kKvHeads, a.num_seqs);
#define PVLC_Q8_LAUNCH(W)                                                                                                   \
    hipLaunchKernelGGL((paged_decode_q8_kernel<W, F32IO, CODE>), grid, dim3((W) * 64), 0, st, p.key_cache, p.value_cache,   \
                       p.exponents, p.cache_lens, p.block_tables, p.uniform_cache_len, p.max_blocks_per_seq, p.num_blocks, \
                       p.partition_tokens | p.max_parts << 16, p)
    switch (q8_waves(launch.partition_tokens)) {
        case 1: PVLC_Q8_LAUNCH(1); break;
        case 2: PVLC_Q8_LAUNCH(2); break;
        case 3: PVLC_Q8_LAUNCH(3); break;
        case 4: PVLC_Q8_LAUNCH(4); break;
        case 6: PVLC_Q8_LAUNCH(6); break;
        case 8: PVLC_Q8_LAUNCH(8); break;
        default: PVLC_Q8_LAUNCH(12); break;
    }
#undef PVLC_Q8_LAUNCH
    return static_cast<int>(hipGetLastError());
}

}  // namespace

int launch_paged_decode_q8(const DecodeLaunch &launch, const DecodeCodes &codes, void *stream) {
    const pvlc_hip_paged_decode_args &a = *launch.args;
    DecodeQ8Params p{};
    p.num_blocks = a.num_blocks;
    p.max_blocks_per_seq = a.max_blocks_per_seq;
    p.block_tables = a.block_tables;
    p.cache_lens = a.cache_lens;
    p.uniform_cache_len = a.uniform_cache_len;
    p.key_cache = a.key_cache;
    p.value_cache = a.value_cache;
    p.exponents = codes.exponents;
    p.query = a.query;
    p.new_key = a.new_key;
    p.new_value = a.new_value;
    p.out = a.out;
    p.rope_cos = a.rope_cos;
    p.rope_sin = a.rope_sin;
    p.rope_rows = a.rope_rows;
    p.positions = a.positions;
    p.rotate_query = a.rotate_query;
    p.partition_tokens = launch.partition_tokens;
    p.max_parts = launch.max_parts;
    p.part_stride = launch.part_stride;
    p.part_o = launch.part_o;
    p.part_ml = launch.part_ml;
    p.counters = launch.counters;
    p.error_word = launch.error_word;
    p.partition_word = launch.partition_word;
    p.scale_log2 = kLog2e / sqrtf(static_cast<float>(kHeadDim));
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (launch.f32) {
        p.query32 = launch.f32->query;
        p.new_key32 = launch.f32->new_key;
        p.new_value32 = launch.f32->new_value;
        p.out32 = launch.f32->out;
        return codes.code == PVLC_HIP_KV_E4M3 ? launch_kernels<true, PVLC_HIP_KV_E4M3>(launch, p, st)
                                              : launch_kernels<true, PVLC_HIP_KV_INT8>(launch, p, st);
    }
    return codes.code == PVLC_HIP_KV_E4M3 ? launch_kernels<false, PVLC_HIP_KV_E4M3>(launch, p, st)
                                          : launch_kernels<false, PVLC_HIP_KV_INT8>(launch, p, st);
}

}  // namespace pvlc
