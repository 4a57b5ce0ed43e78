// Pages of a paged cache: sharing, copying, freeing and compacting, on the
// device and in an order that does not depend on timing.
//
// A pool of num_blocks pages has a reference count for each (how many block
// table entries name it) and a bit for each that is set where the count is 0.
// Fresh pages are the lowest free ones, in the order in which rows and entries
// ask for them; pages that a call frees are free from the next call on.  So the
// work splits into a plan, which one workgroup makes from the rows' lengths and
// the bits (it needs a prefix sum over the rows and a search over the bits, a
// few microseconds), and the execution, which every other workgroup does
// independently: table rows, counts and page copies.
//
// Measured, at 18 layers: four beams of a page (2.4 MB copied): plan 3.8 us,
// execution 3.9, both a chain of rounds; 256 rows (35 MB copied): plan 5.3,
// execution 9.4; 64 sequences compacted, 4600 pages (up to 1.2 GB read and written):
// 168-240 us, at the rate of a large copy.  Copies of 1, 256 and 4000 pages of 8 bits
// (0.3, 76 and 1180 MB read and written): 3.0, 12.8 and 212 us, 5.6 TB/s.  One launch for a small fork, every
// workgroup making the plan by itself and the last one to have it changing the
// counts, took four beams 15.3 us in place of 17.2 for two forks from the host,
// but as long alone, and 24 rows 55 in place of 43: not kept.

#include <hip/hip_runtime.h>

#include <cstdint>

#include "pvlc_device.hpp"
#include "pvlc_internal.hpp"

namespace pvlc {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kWideThreads = 256;
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// Exclusive prefix sum over a workgroup of kThreads; *total receives the sum.
template <int kThreads>
__device__ inline uint32_t plan_scan(uint32_t v, uint32_t *sm, uint32_t *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();  // sm's readers of the scan before are done
    if (lane == 63) sm[wave] = x;
    __syncthreads();
    uint32_t before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) {
        const uint32_t t = sm[w];
        before += w < wave ? t : 0u;
        sum += t;
    }
    *total = sum;
    return before + x - v;
}

__device__ inline bool valid_block(int32_t id, uint32_t num_blocks) { return id >= 0 && static_cast<uint32_t>(id) < num_blocks; }

// Length of row r of the input (a bad one counts as 0).  The sign is looked at
// before the appended rows are added: a fork that found too few pages leaves
// lengths of -1, which one more row does not make an empty sequence.
__device__ inline uint32_t in_length(const PagesFork &f, uint32_t r, uint32_t *errors) {
    const int32_t held = f.lens_in[r];
    const int64_t len = static_cast<int64_t>(held) + f.appended;
    if (held < 0 || len > static_cast<int64_t>(f.max_blocks) * kBlockTokens) {
        *errors |= PVLC_HIP_PAGES_BAD_LENGTH;
        return 0;
    }
    return static_cast<uint32_t>(len);
}

// What becomes of output row r: its parent (-1: none), length, and the blocks it
// needs.
struct RowWant {
    int32_t parent;
    uint32_t length, need;
};
__device__ inline RowWant want_of(const PagesFork &f, uint32_t r, uint32_t *errors) {
    RowWant w{f.parents ? f.parents[r] : (r < f.rows_in ? static_cast<int32_t>(r) : -1), 0, 0};
    int64_t reserve = f.reserve ? f.reserve[r] : static_cast<int64_t>(f.reserve_tokens);
    if (w.parent < -1 || w.parent >= static_cast<int64_t>(f.rows_in)) {
        *errors |= PVLC_HIP_PAGES_BAD_PARENT;
        w.parent = -1;
    }
    if (w.parent >= 0) w.length = in_length(f, static_cast<uint32_t>(w.parent), errors);
    if (reserve < 0) reserve = 0;
    int64_t end = w.length + reserve;
    if (end > static_cast<int64_t>(f.max_blocks) * kBlockTokens) {
        *errors |= PVLC_HIP_PAGES_NO_ROOM;
        end = static_cast<int64_t>(f.max_blocks) * kBlockTokens;
    }
    w.need = static_cast<uint32_t>((end + kBlockTokens - 1) / kBlockTokens);
    return w;
}

// What a row's plan reads: what becomes of it, the entry that it would write next
// and that page's count.
struct RowRead {
    RowWant want;
    int32_t next, count;
};
__device__ inline RowRead read_row(const PagesFork &f, uint32_t r, uint32_t *errors) {
    RowRead row{want_of(f, r, errors), -1, 0};
    const uint32_t filled = row.want.length / kBlockTokens;
    if (row.want.parent >= 0 && row.want.need > filled) {
        row.next = f.tables_in[static_cast<size_t>(row.want.parent) * f.max_blocks + filled];
        if (valid_block(row.next, f.num_blocks)) row.count = f.ref_counts[row.next];
    }
    return row;
}

// The plan of a fork, all that the execution needs of each row in one record.
// An output row keeps the first `kept` of its parent's entries: the filled blocks
// and, for the parent's first child, what follows as far as no other entry names
// it; fresh[base ..] are its others.  Everything of a row stays in LDS and
// registers, and what it needs of the tables is read at once: the launch is a
// chain of rounds through memory (four beams, rows through memory 5.3 us, reads
// where they are needed 4.2, all at once 3.8).  A thread takes a Unit of the mask at a time, bytes
// of pools that have few: it names its pages one after the other.
template <int kThreads, class Unit, uint32_t kUnits>
__global__ __launch_bounds__(kThreads) void pages_fork_plan_kernel(PagesFork f) {
    extern __shared__ uint32_t by_row[];  // first[rows_in], children[rows_in], kept[rows_in]
    __shared__ uint32_t sm[kThreads / 64];
    __shared__ uint32_t sm_errors;
    constexpr uint32_t kBits = sizeof(Unit) * 8, kTile = kThreads * kUnits;  // units of the mask at a time
    // Every pointer in one round of scalar loads.
    asm volatile("" ::"s"(f.parents), "s"(f.reserve), "s"(f.lens_in), "s"(f.tables_in), "s"(f.ref_counts), "s"(f.free_mask), "s"(f.plan.rows),
                 "s"(f.plan.fresh), "s"(f.lens_out));
    uint32_t *first = by_row, *children = first + f.rows_in, *taken = children + f.rows_in;
    const uint32_t i = threadIdx.x;
    if (i == 0) sm_errors = 0;
    for (uint32_t p = i; p < f.rows_in; p += kThreads) {
        first[p] = UINT32_MAX;
        children[p] = 0;
        taken[p] = 0;
    }
    Unit *mask = reinterpret_cast<Unit *>(f.free_mask);  // (little-endian: bit b of unit u is page u * kBits + b)
    const uint32_t units = (f.num_blocks + kBits - 1) / kBits;
    auto load_mask = [&](uint32_t u0, uint32_t (&bits)[kUnits]) {
#pragma unroll
        for (uint32_t k = 0; k < kUnits; ++k) {
            const uint32_t u = u0 + i * kUnits + k;
            bits[k] = u < units ? mask[u] : 0u;
            if (u == units - 1 && f.num_blocks % kBits) bits[k] &= (1u << (f.num_blocks % kBits)) - 1u;
        }
    };
    uint32_t bits[kUnits];
    load_mask(0, bits);  // its use is rounds away
    uint32_t errors = 0, none = 0;
    RowRead mine{};  // of row i, where every row has a thread
    if (i < f.rows_out) mine = read_row(f, i, &errors);
    __syncthreads();
    for (uint32_t r = i; r < f.rows_out; r += kThreads) {
        const int32_t parent = r == i ? mine.want.parent : want_of(f, r, &errors).parent;
        if (parent >= 0) {
            atomicMin(&first[parent], r);
            atomicAdd(&children[parent], 1u);
        }
    }
    __syncthreads();
    uint32_t total = 0;
    for (uint32_t r0 = 0; r0 < f.rows_out; r0 += kThreads) {
        const uint32_t r = r0 + i;
        uint32_t fresh = 0;
        ForkRow row{-1, 0, 0, 0, -1, 0};
        if (r < f.rows_out) {
            const RowRead in = r == i ? mine : read_row(f, r, &none);
            const RowWant &w = in.want;
            const uint32_t filled = w.length / kBlockTokens;
            row = {w.parent, filled, w.need, 0, -1, w.length};
            if (w.parent >= 0 && w.need > filled) {
                int32_t id = in.next, count = in.count;
                if (w.length % kBlockTokens != 0) {
                    row.source = id;
                    if (!valid_block(id, f.num_blocks)) errors |= PVLC_HIP_PAGES_BAD_BLOCK;
                }
                if (!f.keep_inputs && first[w.parent] == r) {
                    while (valid_block(id, f.num_blocks) && count == 1) {
                        if (++row.kept == w.need) break;
                        id = f.tables_in[static_cast<size_t>(w.parent) * f.max_blocks + row.kept];
                        if (valid_block(id, f.num_blocks)) count = f.ref_counts[id];
                    }
                    if (row.kept > filled) row.source = -1;
                    taken[w.parent] = row.kept;
                }
                if (!valid_block(row.source, f.num_blocks)) row.source = -1;
            }
            fresh = w.need - row.kept;
        }
        uint32_t sum;
        row.base = total + plan_scan<kThreads>(fresh, sm, &sum);
        if (r < f.rows_out) f.plan.rows[r] = row;
        total += sum;
    }
    // The lowest `total` free pages.  All free pages up to the last one taken are
    // taken, so the mask is 0 up to the tile that has it; whether there are enough
    // is known when that tile's are counted, before its pages are named.
    uint32_t found = 0, before = 0, u0 = 0;
    bool enough = total == 0;
    while (!enough && u0 < units) {
        if (u0 > 0) load_mask(u0, bits);
        uint32_t here = 0, sum;
#pragma unroll
        for (uint32_t k = 0; k < kUnits; ++k) here += static_cast<uint32_t>(__popc(bits[k]));
        uint32_t at = found + plan_scan<kThreads>(here, sm, &sum);
        before = found;
        found += sum;
        enough = found >= total;
#pragma unroll
        for (uint32_t k = 0; k < kUnits; ++k) {
            uint32_t left = bits[k];
            const uint32_t u = u0 + i * kUnits + k;
            for (; left && at < total; ++at) {
                const int32_t id = static_cast<int32_t>(u * kBits + static_cast<uint32_t>(__ffs(static_cast<int>(left)) - 1));
                left &= left - 1;
                f.plan.fresh[at] = id;
                if (enough) f.ref_counts[id] = 1;
            }
            if (enough && left != bits[k]) mask[u] = static_cast<Unit>(left);
        }
        if (!enough) u0 += kTile;
    }
    if (errors) atomicOr(&sm_errors, errors);
    __syncthreads();
    if (enough && before > 0) {  // pages of the tiles before
        for (uint32_t k = i; k < before; k += kThreads) f.ref_counts[f.plan.fresh[k]] = 1;
        for (uint32_t u = i; u < u0; u += kThreads) mask[u] = 0;
    }
    for (uint32_t p = i; p < f.rows_in; p += kThreads)
        f.plan.inputs[p] = {children[p], in_length(f, p, &none) / kBlockTokens, taken[p], 0};
    for (uint32_t r = i; r < f.rows_out; r += kThreads)
        f.lens_out[r] = enough ? static_cast<int32_t>(r == i ? mine.want.length : f.plan.rows[r].length) : -1;
    if (i == 0) {
        *f.plan.enough = enough;
        const uint32_t e = sm_errors | (enough ? 0u : PVLC_HIP_PAGES_EXHAUSTED);
        if (e) atomicOr(f.plan.error_word, e);
    }
}

// Copies a page of one layer, all planes: the first 8 KiB of each plane (16 bytes
// a thread at a time, 4 where the plane is not made for more) are loaded before
// anything is stored, what is left of larger blocks in a loop.  (Plane by plane
// and piece by piece, each store behind its load, the turnover of 64 sequences took
// 378 us, so 328; with more workgroups, below, 276.)
__device__ inline void copy_pages(const PagePlanes &planes, uint32_t layer, uint32_t src, uint32_t dst) {
    const uint32_t i = threadIdx.x;
    u32x4_t v[kMaxPagePlanes][2];
    const uint8_t *from[kMaxPagePlanes];
    uint8_t *to[kMaxPagePlanes];
#pragma unroll
    for (uint32_t p = 0; p < kMaxPagePlanes; ++p) {
        if (p >= planes.count) continue;
        const PagePlane &q = planes.plane[p];
        to[p] = q.base + q.layer_stride * layer + q.block_bytes * dst;
        from[p] = (q.from ? q.from + q.from_stride * layer : q.base + q.layer_stride * layer) + q.block_bytes * src;
#pragma unroll
        for (uint32_t u = 0; u < 2; ++u) {
            const uint32_t at = i + u * kWideThreads;
            if (q.wide) {
                if (at * 16ull < q.block_bytes) v[p][u] = reinterpret_cast<const u32x4_t *>(from[p])[at];
            } else if (at * 4ull < q.block_bytes) {
                v[p][u][0] = reinterpret_cast<const uint32_t *>(from[p])[at];
            }
        }
    }
#pragma unroll
    for (uint32_t p = 0; p < kMaxPagePlanes; ++p) {
        if (p >= planes.count) continue;
        const PagePlane &q = planes.plane[p];
#pragma unroll
        for (uint32_t u = 0; u < 2; ++u) {
            const uint32_t at = i + u * kWideThreads;
            if (q.wide) {
                if (at * 16ull < q.block_bytes) reinterpret_cast<u32x4_t *>(to[p])[at] = v[p][u];
            } else if (at * 4ull < q.block_bytes) {
                reinterpret_cast<uint32_t *>(to[p])[at] = v[p][u][0];
            }
        }
        if (q.wide) {
            for (uint64_t at = i + 2 * kWideThreads; at < q.block_bytes / 16; at += kWideThreads)
                reinterpret_cast<u32x4_t *>(to[p])[at] = reinterpret_cast<const u32x4_t *>(from[p])[at];
        } else {
            for (uint64_t at = i + 2 * kWideThreads; at < q.block_bytes / 4; at += kWideThreads)
                reinterpret_cast<uint32_t *>(to[p])[at] = reinterpret_cast<const uint32_t *>(from[p])[at];
        }
    }
}

// Workgroups 0 .. rows_in - 1 settle the counts of an input row's pages, the
// next rows_out write an output row's table, the rest copy the page that a row
// writes next, a layer each.
__global__ __launch_bounds__(kWideThreads) void pages_fork_kernel(PagesFork f, PagePlanes planes) {
    const bool enough = *f.plan.enough;
    uint32_t b = blockIdx.x;
    if (b < f.rows_in) {
        const ForkInput in = f.plan.inputs[b];
        if (!enough || (f.keep_inputs && in.children == 0)) return;
        const int32_t *row = f.tables_in + static_cast<size_t>(b) * f.max_blocks;
        uint32_t errors = 0;
        for (uint32_t j = threadIdx.x; j < f.max_blocks; j += kWideThreads) {
            const int32_t id = row[j];
            if (!valid_block(id, f.num_blocks)) {
                if (id != -1 || (in.children && j < in.filled)) errors |= PVLC_HIP_PAGES_BAD_BLOCK;
                continue;
            }
            // an entry is held once by each child that takes it over, and no longer by this row
            const uint32_t held = j < in.filled ? in.children : (j < in.kept ? 1u : 0u);
            const int32_t delta = static_cast<int32_t>(held) - (f.keep_inputs ? 0 : 1);
            if (delta == 0) continue;
            const int32_t old = atomicAdd(&f.ref_counts[id], delta);
            if (old + delta < 0) errors |= PVLC_HIP_PAGES_BAD_COUNT;
            if (old + delta == 0) atomicOr(&f.free_mask[id >> 5], 1u << (id & 31));
        }
        if (errors) atomicOr(f.plan.error_word, errors);
        return;
    }
    b -= f.rows_in;
    if (b < f.rows_out) {
        const ForkRow r = f.plan.rows[b];
        const int32_t *row = f.tables_in + static_cast<size_t>(r.parent < 0 ? 0 : r.parent) * f.max_blocks;
        int32_t *out = f.tables_out + static_cast<size_t>(b) * f.max_blocks;
        for (uint32_t j = threadIdx.x; j < f.max_blocks; j += kWideThreads) {
            int32_t id = -1;
            if (enough && j < r.kept) {
                id = row[j];
                if (!valid_block(id, f.num_blocks)) id = -1;
            } else if (enough && j < r.need) {
                id = f.plan.fresh[r.base + j - r.kept];
            }
            out[j] = id;
        }
        return;
    }
    b -= f.rows_out;
    const ForkRow r = f.plan.rows[b / planes.layers];
    if (!enough || r.source < 0) return;
    copy_pages(planes, b % planes.layers, static_cast<uint32_t>(r.source), static_cast<uint32_t>(f.plan.fresh[r.base]));
}

// Compaction.  With L pages in use, those behind the first L move, in order, to
// the free ones among the first L, in order: the least that moves.
//
// Counts of the words of 32 pages: used_before[w], and L behind the last.
template <int kThreads>
__device__ inline uint32_t count_words(const PagesCompact &c, uint32_t *used_before, uint32_t *sm) {
    const uint32_t words = (c.num_blocks + 31) / 32;
    uint32_t used = 0;
    for (uint32_t w0 = 0; w0 < words; w0 += kThreads) {
        const uint32_t w = w0 + threadIdx.x;
        const uint32_t in_word = w < words ? min(32u, c.num_blocks - w * 32) : 0u;
        uint32_t bits = w < words ? c.free_mask[w] : 0u;
        if (in_word < 32) bits &= (1u << in_word) - 1u;
        uint32_t sum;
        const uint32_t before = plan_scan<kThreads>(in_word - static_cast<uint32_t>(__popc(bits)), sm, &sum);
        if (w < words) used_before[w] = used + before;
        used += sum;
    }
    return used;
}
__global__ __launch_bounds__(kPlanThreads) void pages_count_kernel(PagesCompact c) {
    __shared__ uint32_t sm[kPlanThreads / 64];
    const uint32_t used = count_words<kPlanThreads>(c, c.plan.used_before, sm);
    if (threadIdx.x == 0) c.plan.used_before[(c.num_blocks + 31) / 32] = used;
}

// The list of moves: the k-th used page from L on, to the k-th free page; rank[id]:
// a page's number among them, or -1.  Workgroups of a small pool count its words
// by themselves (a launch of its own for that took 2 us of 38 of a turnover's).
constexpr uint32_t kCountWords = 1024;
template <bool kCounted>
__global__ __launch_bounds__(kWideThreads) void pages_moves_kernel(PagesCompact c) {
    __shared__ uint32_t sm[kWideThreads / 64];
    __shared__ uint32_t sm_before[kCounted ? 1 : kCountWords];
    const uint32_t words = (c.num_blocks + 31) / 32;
    const uint32_t *used_in = kCounted ? c.plan.used_before : sm_before;
    uint32_t live;
    if constexpr (kCounted) {
        live = c.plan.used_before[words];
    } else {
        live = count_words<kWideThreads>(c, sm_before, sm);
        __syncthreads();
        if (blockIdx.x == 0 && threadIdx.x == 0) c.plan.used_before[words] = live;
    }
    const uint32_t id = blockIdx.x * kWideThreads + threadIdx.x;
    if (id >= c.num_blocks) return;
    const uint32_t bit = 1u << (id & 31), bits = c.free_mask[id >> 5];
    const uint32_t used_before = used_in[id >> 5] + static_cast<uint32_t>(__popc(~bits & (bit - 1)));
    const bool free_page = (bits & bit) != 0;
    if (free_page && id < live) c.plan.to[id - used_before] = static_cast<int32_t>(id);
    int32_t rank = -1;
    if (!free_page && id >= live) {
        // its rank among the used pages, less those before L
        const uint32_t lw = live >> 5, below = used_in[lw] + static_cast<uint32_t>(__popc(~c.free_mask[lw] & ((1u << (live & 31)) - 1u)));
        rank = static_cast<int32_t>(used_before - below);
        c.plan.from[rank] = static_cast<int32_t>(id);
    }
    c.plan.rank[id] = rank;
    if (id == live || (live == c.num_blocks && id == 0)) *c.plan.moves = live == c.num_blocks ? 0 : live - used_before;
}

// Copies by (move, layer), then table entries and the caller's map.
__global__ __launch_bounds__(kWideThreads) void pages_compact_kernel(PagesCompact c, PagePlanes planes, uint32_t copy_groups, uint32_t table_groups) {
    const uint32_t moves = *c.plan.moves;
    if (blockIdx.x < copy_groups) {
        const uint64_t items = static_cast<uint64_t>(moves) * planes.layers;
        for (uint64_t item = blockIdx.x; item < items; item += copy_groups) {
            const uint32_t k = static_cast<uint32_t>(item % moves), layer = static_cast<uint32_t>(item / moves);
            const uint32_t src = static_cast<uint32_t>(c.plan.from[k]), dst = static_cast<uint32_t>(c.plan.to[k]);
            copy_pages(planes, layer, src, dst);
            if (layer == 0 && threadIdx.x == 0) {
                c.ref_counts[dst] = c.ref_counts[src];
                c.ref_counts[src] = 0;
            }
        }
        return;
    }
    const uint64_t entries = static_cast<uint64_t>(c.rows) * c.max_blocks, words = (c.num_blocks + 31) / 32;
    const uint32_t live = c.plan.used_before[words];
    const uint64_t stride = static_cast<uint64_t>(table_groups) * kWideThreads, start = static_cast<uint64_t>(blockIdx.x - copy_groups) * kWideThreads + threadIdx.x;
    auto moved = [&](int32_t id) {
        if (!valid_block(id, c.num_blocks)) return id;
        const int32_t k = c.plan.rank[id];
        return k < 0 ? id : c.plan.to[k];
    };
    for (uint64_t e = start; e < entries; e += stride) {
        const int32_t id = c.tables[e], to = moved(id);
        if (to != id) c.tables[e] = to;
    }
    if (c.forward)
        for (uint64_t id = start; id < c.num_blocks; id += stride) c.forward[id] = moved(static_cast<int32_t>(id));
    // the first `live` pages are used (nothing reads the bits in this launch)
    for (uint64_t w = start; w < words; w += stride) {
        const uint64_t first = w * 32;
        uint32_t bits = first >= live ? ~0u : (live - first >= 32 ? 0u : ~0u << (live - first));
        if (c.num_blocks - first < 32) bits &= (1u << (c.num_blocks - first)) - 1u;
        c.free_mask[w] = bits;
    }
}

// Pairs of pages, a (pair, layer) each.
__global__ __launch_bounds__(kWideThreads) void pages_copy_kernel(const int32_t *src, const int32_t *dst, uint32_t src_blocks, uint32_t dst_blocks,
                                                                  PagePlanes planes, uint32_t *error_word) {
    const uint32_t k = blockIdx.x, layer = blockIdx.y;
    const int32_t s = src[k], d = dst[k];
    if (!valid_block(s, src_blocks) || !valid_block(d, dst_blocks)) {
        if (threadIdx.x == 0 && layer == 0 && error_word) atomicOr(error_word, static_cast<uint32_t>(PVLC_HIP_PAGES_BAD_BLOCK));
        return;
    }
    copy_pages(planes, layer, static_cast<uint32_t>(s), static_cast<uint32_t>(d));
}

__global__ __launch_bounds__(kWideThreads) void pages_reset_kernel(int32_t *refs, uint32_t *mask, uint32_t num_blocks, uint32_t *error_word) {
    const uint32_t i = blockIdx.x * kWideThreads + threadIdx.x;
    if (i == 0) *error_word = 0;
    if (i < num_blocks) refs[i] = 0;
    const uint32_t words = (num_blocks + 31) / 32;
    if (i < words) mask[i] = i + 1 == words && (num_blocks & 31) ? (1u << (num_blocks & 31)) - 1u : ~0u;
}

}  // namespace

int launch_pages_reset(int32_t *refs, uint32_t *mask, uint32_t num_blocks, uint32_t *error_word, void *stream) {
    hipLaunchKernelGGL(pages_reset_kernel, dim3((num_blocks + kWideThreads - 1) / kWideThreads), dim3(kWideThreads), 0,
                       static_cast<hipStream_t>(stream), refs, mask, num_blocks, error_word);
    return static_cast<int>(hipGetLastError());
}

int launch_pages_fork(const PagesFork &f, const PagePlanes &planes, void *stream) {
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const uint32_t lds = f.rows_in * 12;
    // A thread for each row and each 8 pages, as far as 1024 go in a few turns,
    // then 32 and 128 pages a thread.
    if (f.rows_in <= 256 && f.rows_out <= 256 && f.num_blocks <= 256 * 8)
        hipLaunchKernelGGL((pages_fork_plan_kernel<256, uint8_t, 1>), dim3(1), dim3(256), lds, st, f);
    else if (f.num_blocks <= 2 * kPlanThreads * 8)
        hipLaunchKernelGGL((pages_fork_plan_kernel<kPlanThreads, uint8_t, 1>), dim3(1), dim3(kPlanThreads), lds, st, f);
    else if (f.num_blocks <= 4 * kPlanThreads * 32)
        hipLaunchKernelGGL((pages_fork_plan_kernel<kPlanThreads, uint32_t, 1>), dim3(1), dim3(kPlanThreads), lds, st, f);
    else
        hipLaunchKernelGGL((pages_fork_plan_kernel<kPlanThreads, uint32_t, 4>), dim3(1), dim3(kPlanThreads), lds, st, f);
    const uint32_t groups = f.rows_in + f.rows_out + f.rows_out * planes.layers;
    hipLaunchKernelGGL(pages_fork_kernel, dim3(groups), dim3(kWideThreads), 0, st, f, planes);
    return static_cast<int>(hipGetLastError());
}

int launch_pages_compact(const PagesCompact &c, const PagePlanes &planes, void *stream) {
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 moves((c.num_blocks + kWideThreads - 1) / kWideThreads);
    if (c.num_blocks <= kCountWords * 32) {
        hipLaunchKernelGGL(pages_moves_kernel<false>, moves, dim3(kWideThreads), 0, st, c);
    } else {
        hipLaunchKernelGGL(pages_count_kernel, dim3(1), dim3(kPlanThreads), 0, st, c);
        hipLaunchKernelGGL(pages_moves_kernel<true>, moves, dim3(kWideThreads), 0, st, c);
    }
    const uint64_t copies = static_cast<uint64_t>(c.num_blocks / 2 + 1) * planes.layers, entries = static_cast<uint64_t>(c.rows) * c.max_blocks + c.num_blocks;
    // (64 sequences' turnover, 4600 pages of 18 layers, with 2048 / 8192 / 16384 /
    // 65536 workgroups: 328 / 288 / 276 / 279 us; non-temporal copies 320 / - / - / -)
    const uint32_t copy_groups = static_cast<uint32_t>(copies < 16384 ? copies : 16384);
    const uint64_t tables = (entries + kWideThreads - 1) / kWideThreads;
    const uint32_t table_groups = static_cast<uint32_t>(tables < 512 ? tables : 512);
    hipLaunchKernelGGL(pages_compact_kernel, dim3(copy_groups + table_groups), dim3(kWideThreads), 0, st, c, planes, copy_groups, table_groups);
    return static_cast<int>(hipGetLastError());
}

int launch_pages_copy(const int32_t *src, const int32_t *dst, uint32_t count, uint32_t src_blocks, uint32_t dst_blocks, const PagePlanes &planes,
                      uint32_t *error_word, void *stream) {
    hipLaunchKernelGGL(pages_copy_kernel, dim3(count, planes.layers), dim3(kWideThreads), 0, static_cast<hipStream_t>(stream), src, dst, src_blocks,
                       dst_blocks, planes, error_word);
    return static_cast<int>(hipGetLastError());
}

}  // namespace pvlc
