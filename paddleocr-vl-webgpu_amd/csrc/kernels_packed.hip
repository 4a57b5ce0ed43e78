// Causal attention of packed prompts: the rows of several sequences, each over
// its own pages (which hold the call's rows by then), behind what these held.
//
//   out_i = sum_j<=i w_ij v_j / sum_j<=i w_ij,  w_ij = exp(q_i k_j / sqrt 128)
//
// 4 * 128 operations a (query, head, key), and with f32 operands 6 * 128, the weights
// being pairs of fp16: large calls are bound by matrix instructions and the vector
// ones between them.  4096 tokens on 61440 rows, all but the loop over whole pieces a
// hundredth of the call, run at 960 TFLOP/s, with f32 operands at 701 (1050 of products); a
// large library product reaches 1090 to 1330.  4 prompts of 4096 to 8192 tokens 627 us (943
// TFLOP/s), 12 of 211 to 2010 tokens 77 (563; items of 18 pieces on average, whose pieces
// would take 47 at the loop's rate: the rest are items' starts and ends, the last round, and
// the append), 6 chunks of 256 to 512 tokens on 16384 rows 201 (576, f32 operands); up to 5%
// more from one card to another.

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "attend_device.hpp"
#include "packed_plan.hpp"

namespace pvlc {
namespace {

typedef float float16_t __attribute__((ext_vector_type(16)));

// Whether the append met values that are not finite in the blocks of an item's rows.
__device__ inline bool item_is_odd(const PackedRows &p, int seq, int begin, int held, int count, int t0) {
    const int32_t *seen = p.odd + first_append_share(p.ragged, seq, begin);
    constexpr int kTokens = kBlockTokens;
    const int before = held / kTokens, a = (held + t0) / kTokens - before, b = (held + min(t0 + kPackedTokens, count) - 1) / kTokens - before;
    return (load_const(seen, a) | load_const(seen, b)) != 0;
}

// A workgroup takes 16 tokens of a sequence and the 8 query heads of a kv head,
// a wave two of the heads: 32 columns, in v_mfma_f32_32x32x16_f16.  Two workgroups
// are on each compute unit, at 188 and 198 registers a wave: one waits or computes
// weights while the other multiplies.  The longest prompts above took 936 us with 64 columns
// a wave straight from the pages, 778 with them through LDS (one wave a SIMD), 749
// with two workgroups of 32, 690 with the plan's order of items, 636 with outputs
// stored through LDS.  The compiler's order of a step is the best one found:
// orders forced by groups ran the loop at 922 to 949 TFLOP/s, other scheduling
// strategies and wave priorities at 933 to 944, where it ran at 955.
constexpr int kWideWaves = 4, kWideStep = 64;
constexpr size_t kPartPairs = kPackedPartPairs / kWideWaves;  // of a wave: (reference, sum) and outputs
constexpr int kStepElems = kWideStep * kHeadDim;  // fp16 elements of a step's keys (or values) of a kv head

template <bool F32>
struct Wide {
    typedef std::conditional_t<F32, float, uint16_t> Element;
    const PackedRows &p;
    const uint32_t g;
    const int lane, col, half, wave;
    half8_t qf[8];
    float16_t o[4];  // dims dt * 32 + (r / 4) * 8 + half * 4 + r % 4 of the lane's query
    float m, l;
    int limit;

    __device__ Wide(const PackedRows &rows, uint32_t head)
        : p(rows), g(head), lane(threadIdx.x & 63), col(lane & 31), half(lane >> 5),
          wave(__builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6))) {}

    // The query of this lane's column (past the sequence: its last one again, not
    // stored): sent for, then rotated.
    AttendQuery<F32> raw[4];
    int64_t pos;
    __device__ __attribute__((always_inline)) void send_for_queries(const PackedItem &q) {
        const int t = min(q.t0 + (col & 15), q.count - 1);
        const int64_t at = q.begin + static_cast<int64_t>(t);
        limit = q.held + t + 1;
        pos = p.positions ? p.positions[at] : q.held + static_cast<int64_t>(t);
        const Element *src = static_cast<const Element *>(p.query) + at * p.query_stride + (g * kGroup + wave * 2 + (col >> 4)) * kHeadDim;
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) raw[kb].load(src, kb * 16 + half * 8);
    }
    __device__ __attribute__((always_inline)) void take_queries() {
        const bool rope = p.rope_cos != nullptr && pos >= 0 && pos < static_cast<int64_t>(p.rope_rows);
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
            float4_t cs[2]{}, sn[2]{};
            if (rope) {
#pragma unroll
                for (int f = 0; f < 2; ++f) {
                    cs[f] = *reinterpret_cast<const float4_t *>(p.rope_cos + pos * 64 + kb * 16 + half * 8 + f * 4);
                    sn[f] = *reinterpret_cast<const float4_t *>(p.rope_sin + pos * 64 + kb * 16 + half * 8 + f * 4);
                }
            }
            raw[kb].rotate(rope, cs, sn, &qf[kb], &qf[kb + 4]);
        }
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;
    }

    // S^T = K Q^T of 32 keys: a row of the first operand is a slot of a block, so
    // lane (query, half) receives keys half * 8 + 0 .. 7 of each of the two
    // blocks in order, which is its operand of the second product.
    typedef float16_t Scores;
    __device__ __attribute__((always_inline)) void scores(const uint16_t *kl, Scores &x) const {
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = 0.f;
        const uint16_t *src = kl + (col >> 4) * static_cast<int>(kBlockHeadElems) + half * 128 + (col & 15) * 8;
#pragma unroll
        for (int kb = 0; kb < 8; ++kb) {
            const half8_t k = *reinterpret_cast<const half8_t *>(src + kb * 256);
            x = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qf[kb], x, 0, 0, 0);
        }
    }
    __device__ __attribute__((always_inline)) void mask(int key0, Scores &x) const {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int key = key0 + (r >> 3) * 16 + half * 8 + (r & 7);
            x[r] = key < limit ? x[r] : -INFINITY;
        }
    }
    // The softmax reference moves when a maximum passes it by 2^8 or more.
    __device__ __attribute__((always_inline)) void rescale(const Scores &x) {
        float c = m;
#pragma unroll
        for (int r = 0; r < 16; ++r) c = fmaxf(c, x[r]);
        const attend_u32x2 v = __builtin_amdgcn_permlane32_swap(__float_as_uint(c), __float_as_uint(c), false, false);
        const float top = fmaxf(__uint_as_float(v[0]), __uint_as_float(v[1]));
        if (__any((top - m) * p.scale_log2 > kAttendRescaleLog2)) {  // uniform
            const float a = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - top) * p.scale_log2);
            m = top;
            l *= a;
#pragma unroll
            for (int dt = 0; dt < 4; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[dt][r] *= a;
        }
    }
    // The values that are not finite, of a key in `block`, where the query sees it.
    __device__ __attribute__((always_inline)) void add_odd(const uint16_t *block, int key) {
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                if ((r & 3) == 0) __builtin_amdgcn_sched_barrier(0);  // (few loads at once: seldom run, and must not cost the loop registers)
                const int d = dt * 32 + (r >> 2) * 8 + half * 4 + (r & 3);
                o[dt][r] += odd_value(block[d * static_cast<int>(kBlockTokens) + key % static_cast<int>(kBlockTokens)], key < limit);
            }
    }
    // The weights of 32 keys in fp16 (with f32 operands as hi + lo), their sum as
    // rounded, and O^T += V^T P^T.
    __device__ __attribute__((always_inline)) void product(const Scores &x, const uint16_t *vl) {
        const half2_t ones = {static_cast<_Float16>(1.0f), static_cast<_Float16>(1.0f)};
        half8_t hi[2], lo[2];
        const float ms = m == -INFINITY ? 0.f : m * p.scale_log2;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(x[b * 8 + e], p.scale_log2, -ms));
                hi[b][e] = to_h(w);
                if constexpr (F32) lo[b][e] = to_h(w - static_cast<float>(hi[b][e]));
            }
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                l = __builtin_amdgcn_fdot2(half2_t{hi[b][e], hi[b][e + 1]}, ones, l, false);
                if constexpr (F32) l = __builtin_amdgcn_fdot2(half2_t{lo[b][e], lo[b][e + 1]}, ones, l, false);
            }
        }
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int dt = 0; dt < 4; ++dt) {
                const half8_t v = *reinterpret_cast<const half8_t *>(vl + (b * 2 + half) * (static_cast<int>(kHeadDim) * 8) + (dt * 32 + col) * 8);
                o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, hi[b], o[dt], 0, 0, 0);
                if constexpr (F32) o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, lo[b], o[dt], 0, 0, 0);
            }
    }
    // A part of the keys, left as it is, and the parts of an item joined in their
    // order: wave and lane hold there what they hold here.  Relaxed agent-scope
    // accesses, coherent across the XCDs' L2s by themselves (a fence at that scope
    // would write the whole L2 back).
    __device__ uint64_t *part(int slot) const { return p.partials + ((static_cast<size_t>(slot) * 2 + g) * kWideWaves + wave) * kPartPairs + lane; }
    static __device__ uint64_t pair(float a, float b) { return static_cast<uint64_t>(__float_as_uint(a)) | static_cast<uint64_t>(__float_as_uint(b)) << 32; }
    __device__ void leave(int slot) const {
        uint64_t *to = part(slot);
        __hip_atomic_store(to, pair(m, l), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
        for (int i = 0; i < 32; ++i)
            __hip_atomic_store(to + (i + 1) * 64, pair(o[i >> 3][(i & 7) * 2], o[i >> 3][(i & 7) * 2 + 1]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __device__ void join(const PackedItem &q) {
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;
        for (int s = q.slots; s < q.slots + q.parts; ++s) {
            const uint64_t *from = part(s);
            uint64_t in[33];
#pragma unroll
            for (int i = 0; i < 33; ++i) in[i] = __hip_atomic_load(from + i * 64, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            auto low = [&](int i) { return __uint_as_float(static_cast<uint32_t>(in[i])); };
            auto high = [&](int i) { return __uint_as_float(static_cast<uint32_t>(in[i] >> 32)); };
            const float n = low(0), top = fmaxf(m, n);
            const float a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - top) * p.scale_log2);
            const float c = n == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((n - top) * p.scale_log2);
            l = l * a + high(0) * c;
            m = top;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                float16_t &t = o[i >> 3];
                t[(i & 7) * 2] = t[(i & 7) * 2] * a + low(i + 1) * c;
                t[(i & 7) * 2 + 1] = t[(i & 7) * 2 + 1] * a + high(i + 1) * c;
            }
        }
    }
    // 1 / the sum of the query's weights, over both halves of the wave.
    __device__ float inverse_sum() const {
        const attend_u32x2 v = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
        return 1.0f / (__uint_as_float(v[0]) + __uint_as_float(v[1]));
    }
    // The wave's outputs, turned in LDS (16 KiB of its own) so that 16 lanes store
    // a row of 128 dims, or half of one in f32: whole lines.
    __device__ void store(const PackedItem &q, float inv, void *own) const {
        constexpr int kPasses = F32 ? 2 : 1, kDims = kHeadDim / kPasses, kPitch = kDims + 16 / sizeof(Element), kPer = 16 / sizeof(Element);
        Element *lds = static_cast<Element *>(own);
        typedef std::conditional_t<F32, float4_t, half4_t> Four;
#pragma unroll
        for (int pass = 0; pass < kPasses; ++pass) {
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int dt = 0; dt < 4 / kPasses; ++dt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float16_t &from = o[pass * (4 / kPasses) + dt];
                    Four f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if constexpr (F32) f[e] = from[r * 4 + e] * inv;
                        else f[e] = to_h(from[r * 4 + e] * inv);
                    }
                    *reinterpret_cast<Four *>(lds + col * kPitch + dt * 32 + r * 8 + half * 4) = f;
                }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int c = i * 4 + (lane >> 4), t = q.t0 + (c & 15), d = (lane & 15) * kPer;
                const q8x4_t v = *reinterpret_cast<const q8x4_t *>(lds + c * kPitch + d);
                if (t < q.count)
                    *reinterpret_cast<q8x4_t *>(static_cast<Element *>(p.out) +
                                                ((q.begin + static_cast<int64_t>(t)) * kQueryHeads + g * kGroup + wave * 2 + (c >> 4)) * kHeadDim +
                                                pass * kDims + d) = v;
            }
        }
    }
};

// Double-buffered LDS, filled by direct global-to-LDS loads (lane l's 16 bytes
// land at the wave's base + 16 l): wave w fetches the step's block w, keys in
// their own order, values as [token half][128 dims][8 tokens], so that every 16
// lanes of an operand's read are 256 contiguous bytes.
template <bool F32>
__global__ __launch_bounds__(kWideWaves * 64, 2) void packed_wide_kernel(PackedRows p) {
    // (distinct arrays, picked at compile time, so that the compiler sees that a
    // step's loads and its reads touch different ones)
    __shared__ __align__(16) uint16_t sk0[kStepElems], sk1[kStepElems], sv0[kStepElems], sv1[kStepElems];
    __shared__ int sm_last;
    const uint32_t g = blockIdx.x & 1u, b = blockIdx.x >> 1;
    PackedItem q;
    if (p.items) {
        const uint32_t items = load_const(p.count, 0);
        q = load_item(p.items, b);  // (beside the count, in one round)
        if (b >= items) return;
    } else {
        const SeqRows s = find_share<kPackedTokens, 1>(p.ragged, (gridDim.x >> 1) - 1 - b);
        if (!s.ok || s.share >= (s.count + kPackedTokens - 1) / kPackedTokens) return;  // (the append reports it)
        q = packed_item(s);
    }
    Wide<F32> w(p, g);
    const int lane = w.lane, wave = w.wave, t0 = q.t0, first = q.first, end = q.end;
    const int valid = q.held + q.count, last_tile = (min(q.held + t0 + kPackedTokens, valid) - 1) >> 4;
    const int masked = (q.held + t0 + 1) / 32;  // pieces from this one on reach past the first query's keys
    const bool odd = item_is_odd(p, q.seq, q.begin, q.held, q.count, t0);

    const int32_t *table = p.ragged.tables ? p.ragged.tables + static_cast<size_t>(q.seq) * p.ragged.max_blocks : nullptr;
    const int64_t base = static_cast<int64_t>(q.seq) * p.ragged.max_blocks;
    bool bad = false;  // uniform over the wave: a block id outside the planes
    auto slab = [&](int tile) -> size_t {
        tile = min(tile, last_tile);  // (tiles behind the last are never used)
        const int64_t id = table ? load_const(table, tile) : base + tile;
        const bool ok = id >= 0 && id < static_cast<int64_t>(p.ragged.num_blocks);
        bad |= !ok;
        return (static_cast<size_t>(ok ? id : 0) * kKvHeads + g) * kBlockHeadElems;
    };
    typedef __attribute__((address_space(3))) void *lds_ptr;
    // A step is pieces n and n + 1: their values, and the keys of pieces n + 1 and n + 2.
    auto fetch_k = [&](int n, uint16_t *dst) {
        const uint16_t *src = p.key_cache + slab(n * 2 + 2 + wave) + lane * 8;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            __builtin_amdgcn_global_load_lds(src + r * 512, (lds_ptr)(dst + wave * static_cast<int>(kBlockHeadElems) + r * 512), 16, 0, 0);
    };
    auto fetch_v = [&](int n, uint16_t *dst) {
        const uint16_t *src = p.value_cache + slab(n * 2 + wave) + lane * 16;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            __builtin_amdgcn_global_load_lds(src + (r & 1) * 1024 + (r >> 1) * 8, (lds_ptr)(dst + wave * static_cast<int>(kBlockHeadElems) + r * 512), 16, 0, 0);
    };
    constexpr int kPiece = kStepElems / 2;
    w.send_for_queries(q);
    fetch_k(first - 1, sk1);  // (of which the first piece's are read)
    fetch_k(first, sk0);
    fetch_v(first, sv0);
    w.take_queries();
    __syncthreads();  // (every wave waits for its loads first)

    typename Wide<F32>::Scores x, y;
    w.scores(sk1, x);
    if (masked <= first) w.mask(first * 32, x);
    w.rescale(x);
    __syncthreads();
    // The scores of a piece stand beside the weights of the one before, its
    // maxima beside that one's product.
    auto plain = [&](int n, const uint16_t *kc, uint16_t *kn, const uint16_t *vc, uint16_t *vn) __attribute__((always_inline)) {
        fetch_k(n + 2, kn);
        fetch_v(n + 2, vn);
        w.scores(kc, y);
        w.product(x, vc);
        w.rescale(y);
        w.scores(kc + kPiece, x);
        w.product(y, vc + kPiece);
        w.rescale(x);
        __syncthreads();
    };
    auto edge = [&](int n, const uint16_t *kc, uint16_t *kn, uint16_t *vc, uint16_t *vn) __attribute__((always_inline)) {
        fetch_k(n + 2, kn);
        fetch_v(n + 2, vn);
        if ((n + 2) * 32 > valid || odd) {
            // Values behind the sequence's rows become 0: what the pages hold there may
            // be NaN, and a weight of 0 would not remove it.  And values of the
            // item's own rows that are not finite: some of its queries do not see them.
            for (int i = static_cast<int>(threadIdx.x); i < kStepElems; i += kWideWaves * 64)
                if (n * 32 + (i >> 11) * 16 + ((i >> 10) & 1) * 8 + (i & 7) >= valid || (odd && is_odd(vc[i]))) vc[i] = 0;
            __syncthreads();
        }
        if (n + 1 < end) {
            w.scores(kc, y);
            if (masked <= n + 1) w.mask((n + 1) * 32, y);
        }
        w.product(x, vc);
        if (n + 1 < end) {
            w.rescale(y);
            if (n + 2 < end) {
                w.scores(kc + kPiece, x);
                if (masked <= n + 2) w.mask((n + 2) * 32, x);
            }
            w.product(y, vc + kPiece);
            if (n + 2 < end) w.rescale(x);
        }
        __syncthreads();
    };
    int n = first;
    for (; n + 4 < min(masked, end); n += 4) {
        plain(n, sk0, sk1, sv0, sv1);
        plain(n + 2, sk1, sk0, sv1, sv0);
    }
    const int edges = n;
    for (; n < end; n += 4) {
        edge(n, sk0, sk1, sv0, sv1);
        if (n + 2 < end) edge(n + 2, sk1, sk0, sv1, sv0);
    }
    if (odd) {  // uniform
#pragma unroll 1
        for (int key = edges * 32; key < min(end * 32, valid) && key / static_cast<int>(kBlockTokens) <= last_tile; ++key)
            w.add_odd(p.value_cache + slab(key / static_cast<int>(kBlockTokens)), key);
    }

    if (bad && lane == 0) atomicOr(p.error_word, 2u);

    if (q.slot >= 0) {
        // A part of the keys.  The workgroup that leaves the last one of its item joins
        // them (a launch of its own would take calls without parts 1 us, too).
        w.leave(q.slot);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the wave's part is there
        __syncthreads();
        if (threadIdx.x == 0)
            sm_last = __hip_atomic_fetch_add(p.arrived + q.slots * 2 + static_cast<int>(g), 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == static_cast<uint32_t>(q.parts) - 1;
        __syncthreads();
        if (!sm_last) return;  // uniform
        w.join(q);
    }
    // (every wave is past its last read of the buffers)
    w.store(q, w.inverse_sum(), wave < 2 ? (wave == 0 ? sk0 : sk1) : (wave == 2 ? sv0 : sv1));
}

// Small calls: a workgroup takes 16 tokens and one head, its waves the pieces of
// 32 keys in turn, keys and values from the pages into registers; no plan.  More
// workgroups, and each has a quarter of the steps, but every head reads the keys
// and values again.
constexpr int kNarrowWaves = 4;
template <bool F32>
__global__ __launch_bounds__(kNarrowWaves * 64, 2) void packed_narrow_kernel(PackedRows p) {
    constexpr int kF16 = PVLC_HIP_KV_F16, kThreads = kNarrowWaves * 64;
    typedef typename AttendQuery<F32>::Element Element;
    __shared__ float sm_m[kNarrowWaves][16], sm_l[kNarrowWaves][16];
    __shared__ float4_t sm_o[kNarrowWaves][8 * 64];
    const uint32_t g = blockIdx.x & 1u, head = g * kGroup + ((blockIdx.x >> 1) & (kGroup - 1));
    const SeqRows q = find_share<kPackedTokens, 1>(p.ragged, blockIdx.x / kQueryHeads);
    const int t0 = q.share * kPackedTokens;
    if (!q.ok || t0 >= q.count) return;  // uniform (the append reports it)
    const int lane = threadIdx.x & 63, row = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int valid = q.held + q.count, keys = min(q.held + t0 + kPackedTokens, valid);
    // Waves 0 and 1 rotate a pair of 32-dim slices each; all take the queries from LDS.
    const int t = min(t0 + row, q.count - 1);  // (past the sequence: its last one again, not stored)
    AttendQuery<F32> raw;
    float4_t cs[2]{}, sn[2]{};
    bool rope = false;
    if (wave < 2) {
        const int64_t at = q.begin + static_cast<int64_t>(t), pos = p.positions ? p.positions[at] : q.held + static_cast<int64_t>(t);
        raw.load(static_cast<const Element *>(p.query) + at * p.query_stride + head * kHeadDim, attend_dim<kF16>(wave, kg));
        rope = p.rope_cos != nullptr && pos >= 0 && pos < static_cast<int64_t>(p.rope_rows);
        if (rope) {
#pragma unroll
            for (int f = 0; f < 2; ++f) {
                cs[f] = *reinterpret_cast<const float4_t *>(p.rope_cos + pos * 64 + attend_dim<kF16>(wave, kg) + f * 4);
                sn[f] = *reinterpret_cast<const float4_t *>(p.rope_sin + pos * 64 + attend_dim<kF16>(wave, kg) + f * 4);
            }
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    AttendPages pages;
    pages.keys = reinterpret_cast<const uint8_t *>(p.key_cache);
    pages.values = reinterpret_cast<const uint8_t *>(p.value_cache);
    pages.exponents = nullptr;
    pages.table = p.ragged.tables ? p.ragged.tables + static_cast<size_t>(q.seq) * p.ragged.max_blocks : nullptr;
    pages.first = static_cast<uint32_t>(q.seq) * p.ragged.max_blocks;
    pages.num_blocks = p.ragged.num_blocks;
    pages.head = g;
    pages.last_tile = (keys - 1) >> 4;
    Attend<kF16, F32, 1, true> loop;
    loop.begin(pages, wave, (keys + kAttendStep - 1) / kAttendStep, kNarrowWaves);
    loop.odd = item_is_odd(p, q.seq, q.begin, q.held, q.count, t0);
    half8_t *const sm_q = reinterpret_cast<half8_t *>(&sm_o[0][0]);  // [kb][lane], before the join
    if (wave < 2) {
        half8_t lo, hi;
        raw.rotate(rope, cs, sn, &lo, &hi);
        sm_q[wave * 64 + lane] = lo;
        sm_q[(wave + 2) * 64 + lane] = hi;
    }
    // (fences of LDS alone: the keys and values stay in flight)
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    half8_t qf[1][4];
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) qf[0][kb] = sm_q[kb * 64 + lane];
    const int limit[1] = {q.held + t + 1};
    AttendState<1> st;
    st.clear();
    const int masked = (q.held + t0 + 1) / kAttendStep;
    loop.run(qf, masked, limit, valid, p.scale_log2, st);
    if (loop.bad && lane == 0) atomicOr(p.error_word, 2u);
    if (loop.odd) loop.add_odd(masked, limit, valid, st);
    const float l = column_sum(st.l[0]);
    if (kg == 0) {
        sm_m[wave][row] = st.m[0];
        sm_l[wave][row] = l;
    }
    __syncthreads();
    float m = sm_m[0][row], sum = 0.f;
#pragma unroll
    for (int w = 1; w < kNarrowWaves; ++w) m = fmaxf(m, sm_m[w][row]);
#pragma unroll
    for (int w = 0; w < kNarrowWaves; ++w) sum += sm_l[w][row] * (sm_m[w][row] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((sm_m[w][row] - m) * p.scale_log2));
    const float a = st.m[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((st.m[0] - m) * p.scale_log2), factor = a * (1.0f / sum);
#pragma unroll
    for (int c = 0; c < 8; ++c) sm_o[wave][c * 64 + lane] = st.o[0][c] * factor;
    __syncthreads();
#pragma unroll
    for (int i = static_cast<int>(threadIdx.x); i < 8 * 64; i += kThreads) {
        const int token = t0 + (i & 15), d = (i >> 6) * 16 + ((i >> 4) & 3) * 4;
        float4_t v = sm_o[0][i];
#pragma unroll
        for (int w = 1; w < kNarrowWaves; ++w) v += sm_o[w][i];
        if (token < q.count) {
            Element *dst = static_cast<Element *>(p.out) + ((q.begin + static_cast<int64_t>(token)) * kQueryHeads + head) * kHeadDim + d;
            if constexpr (F32) *reinterpret_cast<float4_t *>(dst) = v;
            else *reinterpret_cast<half4_t *>(dst) = half4_t{to_h(v[0]), to_h(v[1]), to_h(v[2]), to_h(v[3])};
        }
    }
}

}  // namespace

int launch_packed_prefill(const PackedRows &rows, void *stream) {
    PackedRows p = rows;
    p.scale_log2 = kAttendLog2e / sqrtf(static_cast<float>(kHeadDim));
    const auto st = static_cast<hipStream_t>(stream);
    if (p.narrow) {
        const RaggedRows &r = p.ragged;
        const uint32_t shares = r.offsets ? r.rows / kPackedTokens + r.num_seqs : r.num_seqs * shares_of_each<kPackedTokens, 1>(r.each);
        hipLaunchKernelGGL(p.f32 ? packed_narrow_kernel<true> : packed_narrow_kernel<false>, dim3(kQueryHeads * shares), dim3(kNarrowWaves * 64), 0, st, p);
        return static_cast<int>(hipGetLastError());
    }
    hipLaunchKernelGGL(p.f32 ? packed_wide_kernel<true> : packed_wide_kernel<false>, dim3(2 * p.max_items), dim3(kWideWaves * 64), 0, st, p);
    return static_cast<int>(hipGetLastError());
}

}  // namespace pvlc
