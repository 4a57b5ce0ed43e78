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

#include <hip/hip_runtime.h>

#include <cstdint>

#include "pvlc_device.hpp"
#include "pvlc_internal.hpp"

namespace pvlc {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kWideThreads = 256;
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// Exclusive prefix sum over a workgroup of kPlanThreads; *total receives the sum.
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
    for (int w = 0; w < kPlanThreads / 64; ++w) {
        const uint32_t t = sm[w];
        before += w < wave ? t : 0u;
        sum += t;
    }
    *total = sum;
    return before + x - v;
}

__device__ inline bool valid_block(int32_t id, uint32_t num_blocks) { return id >= 0 && static_cast<uint32_t>(id) < num_blocks; }

// Length of row r of the input, and whether it is one (a bad one counts as 0).
__device__ inline uint32_t in_length(const PagesFork &f, uint32_t r, bool *bad) {
    const int64_t len = static_cast<int64_t>(f.lens_in[r]) + f.appended;
    if (len < 0 || len > static_cast<int64_t>(f.max_blocks) * kBlockTokens) {
        *bad = true;
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
    if (w.parent < -1 || w.parent >= static_cast<int64_t>(f.rows_in)) {
        *errors |= PVLC_HIP_PAGES_BAD_PARENT;
        w.parent = -1;
    }
    if (w.parent >= 0) {
        bool bad = false;
        w.length = in_length(f, static_cast<uint32_t>(w.parent), &bad);
        if (bad) *errors |= PVLC_HIP_PAGES_BAD_LENGTH;
    }
    int64_t reserve = f.reserve ? f.reserve[r] : static_cast<int64_t>(f.reserve_tokens);
    if (reserve < 0) reserve = 0;
    int64_t end = w.length + reserve;
    if (end > static_cast<int64_t>(f.max_blocks) * kBlockTokens) {
        *errors |= PVLC_HIP_PAGES_NO_ROOM;
        end = static_cast<int64_t>(f.max_blocks) * kBlockTokens;
    }
    w.need = static_cast<uint32_t>((end + kBlockTokens - 1) / kBlockTokens);
    return w;
}

// The plan of a fork.  kept[r]: entries of row r taken over from its parent (the
// filled blocks, and behind them what the parent's first child may write itself:
// pages that nobody else names); fresh[base[r]..]: its others.  first[p]: the
// lowest row with parent p; children[p]: how many there are.
__global__ __launch_bounds__(kPlanThreads) void pages_fork_plan_kernel(PagesFork f) {
    __shared__ uint32_t sm[kPlanThreads / 64];
    __shared__ uint32_t sm_errors;
    const uint32_t i = threadIdx.x;
    if (i == 0) sm_errors = 0;
    for (uint32_t p = i; p < f.rows_in; p += kPlanThreads) {
        f.plan.first[p] = UINT32_MAX;
        f.plan.children[p] = 0;
    }
    __threadfence_block();
    __syncthreads();
    uint32_t errors = 0;
    for (uint32_t r = i; r < f.rows_out; r += kPlanThreads) {
        const RowWant w = want_of(f, r, &errors);
        if (w.parent >= 0) {
            atomicMin(&f.plan.first[w.parent], r);
            atomicAdd(&f.plan.children[w.parent], 1u);
        }
    }
    __threadfence_block();
    __syncthreads();
    uint32_t total = 0;
    for (uint32_t r0 = 0; r0 < f.rows_out; r0 += kPlanThreads) {
        const uint32_t r = r0 + i;
        uint32_t fresh = 0;
        if (r < f.rows_out) {
            uint32_t none = 0;
            const RowWant w = want_of(f, r, &none);
            uint32_t kept = 0;
            if (w.parent >= 0) {
                kept = w.length / kBlockTokens;  // filled blocks are shared
                if (!f.keep_inputs && __hip_atomic_load(&f.plan.first[w.parent], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == r) {
                    const int32_t *row = f.tables_in + static_cast<size_t>(w.parent) * f.max_blocks;
                    while (kept < w.need) {
                        const int32_t id = row[kept];
                        if (!valid_block(id, f.num_blocks) || f.ref_counts[id] != 1) break;
                        ++kept;
                    }
                }
            }
            kept = min(kept, w.need);
            fresh = w.need - kept;
            f.plan.kept[r] = kept;
        }
        uint32_t sum;
        const uint32_t base = total + plan_scan(fresh, sm, &sum);
        if (r < f.rows_out) f.plan.base[r] = base;
        total += sum;
    }
    // The lowest `total` free pages.
    const uint32_t words = (f.num_blocks + 31) / 32;
    uint32_t found = 0;
    for (uint32_t w0 = 0; w0 < words && found < total; w0 += kPlanThreads) {
        const uint32_t w = w0 + i;
        uint32_t bits = w < words ? f.free_mask[w] : 0u;
        if (w == words - 1 && (f.num_blocks & 31)) bits &= (1u << (f.num_blocks & 31)) - 1u;
        uint32_t sum;
        uint32_t at = found + plan_scan(static_cast<uint32_t>(__popc(bits)), sm, &sum);
        for (; bits && at < total; ++at) {
            f.plan.fresh[at] = static_cast<int32_t>(w * 32 + static_cast<uint32_t>(__ffs(bits) - 1));
            bits &= bits - 1;
        }
        found += sum;
    }
    if (errors) atomicOr(&sm_errors, errors);
    __threadfence_block();
    __syncthreads();
    const bool enough = found >= total;  // uniform
    if (enough)
        for (uint32_t k = i; k < total; k += kPlanThreads) {
            const int32_t id = f.plan.fresh[k];
            f.ref_counts[id] = 1;
            atomicAnd(&f.free_mask[id >> 5], ~(1u << (id & 31)));
        }
    if (i == 0) {
        *f.plan.enough = enough;
        const uint32_t e = sm_errors | (enough ? 0u : PVLC_HIP_PAGES_EXHAUSTED);
        if (e) atomicOr(f.plan.error_word, e);
    }
}

// Copies bytes of one page of a plane (a multiple of 4 bytes; 16-byte pieces
// where size and planes allow it).
__device__ inline void copy_page(const uint8_t *src, uint8_t *dst, uint64_t bytes, bool wide, uint32_t thread, uint32_t threads) {
    if (wide) {
        for (uint64_t at = thread; at < bytes / 16; at += threads)
            reinterpret_cast<u32x4_t *>(dst)[at] = reinterpret_cast<const u32x4_t *>(src)[at];
    } else {
        for (uint64_t at = thread; at < bytes / 4; at += threads)
            reinterpret_cast<uint32_t *>(dst)[at] = reinterpret_cast<const uint32_t *>(src)[at];
    }
}

__device__ inline void copy_pages(const PagePlanes &planes, uint32_t layer, uint32_t src, uint32_t dst) {
#pragma unroll
    for (uint32_t p = 0; p < kMaxPagePlanes; ++p) {
        if (p >= planes.count) break;
        uint8_t *base = planes.plane[p].base + planes.plane[p].layer_stride * layer;
        const uint8_t *from = planes.plane[p].from ? planes.plane[p].from + planes.plane[p].from_stride * layer : base;
        copy_page(from + planes.plane[p].block_bytes * src, base + planes.plane[p].block_bytes * dst, planes.plane[p].block_bytes,
                  planes.plane[p].wide, threadIdx.x, kWideThreads);
    }
}

// Workgroups 0 .. rows_in - 1 settle the counts of an input row's pages, the
// next rows_out write an output row's table, the rest copy the page that a row
// writes next, a layer each.
__global__ __launch_bounds__(kWideThreads) void pages_fork_kernel(PagesFork f, PagePlanes planes) {
    const bool enough = *f.plan.enough;
    uint32_t b = blockIdx.x;
    if (b < f.rows_in) {
        if (!enough) return;
        const uint32_t children = f.plan.children[b];
        if (f.keep_inputs && children == 0) return;
        bool bad = false;
        const uint32_t filled = in_length(f, b, &bad) / kBlockTokens, first = f.plan.first[b];
        const uint32_t kept = !f.keep_inputs && first != UINT32_MAX ? f.plan.kept[first] : 0u;
        const int32_t *row = f.tables_in + static_cast<size_t>(b) * f.max_blocks;
        uint32_t errors = 0;
        for (uint32_t j = threadIdx.x; j < f.max_blocks; j += kWideThreads) {
            const int32_t id = row[j];
            if (!valid_block(id, f.num_blocks)) {
                if (id != -1 || (children && j < filled)) errors |= PVLC_HIP_PAGES_BAD_BLOCK;
                continue;
            }
            // an entry is held once by each child that takes it over, and no longer by this row
            uint32_t held = j < filled ? children : (j < kept ? 1u : 0u);
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
    uint32_t none = 0;
    if (b < f.rows_out) {
        const RowWant w = want_of(f, b, &none);
        const uint32_t kept = f.plan.kept[b], base = f.plan.base[b];
        const int32_t *row = f.tables_in + static_cast<size_t>(w.parent < 0 ? 0 : w.parent) * f.max_blocks;
        int32_t *out = f.tables_out + static_cast<size_t>(b) * f.max_blocks;
        for (uint32_t j = threadIdx.x; j < f.max_blocks; j += kWideThreads) {
            int32_t id = -1;
            if (enough && j < kept) {
                id = row[j];
                if (!valid_block(id, f.num_blocks)) id = -1;
            } else if (enough && j < w.need) {
                id = f.plan.fresh[base + j - kept];
            }
            out[j] = id;
        }
        if (threadIdx.x == 0) f.lens_out[b] = enough ? static_cast<int32_t>(w.length) : -1;
        return;
    }
    b -= f.rows_out;
    if (!enough) return;
    const uint32_t r = b / planes.layers, layer = b % planes.layers;
    const RowWant w = want_of(f, r, &none);
    const uint32_t filled = w.length / kBlockTokens;
    if (w.parent < 0 || w.length % kBlockTokens == 0 || f.plan.kept[r] > filled) return;  // (kept >= filled)
    const int32_t src = f.tables_in[static_cast<size_t>(w.parent) * f.max_blocks + filled];
    if (!valid_block(src, f.num_blocks)) {
        if (threadIdx.x == 0) atomicOr(f.plan.error_word, static_cast<uint32_t>(PVLC_HIP_PAGES_BAD_BLOCK));
        return;
    }
    copy_pages(planes, layer, static_cast<uint32_t>(src), static_cast<uint32_t>(f.plan.fresh[f.plan.base[r]]));
}

// Compaction.  With L pages in use, those behind the first L move, in order, to
// the free ones among the first L, in order: the least that moves.
//
// Counts of the words of 32 pages: used_before[w], and L behind the last.
__global__ __launch_bounds__(kPlanThreads) void pages_count_kernel(PagesCompact c) {
    __shared__ uint32_t sm[kPlanThreads / 64];
    const uint32_t words = (c.num_blocks + 31) / 32;
    uint32_t used = 0;
    for (uint32_t w0 = 0; w0 < words; w0 += kPlanThreads) {
        const uint32_t w = w0 + threadIdx.x;
        const uint32_t in_word = w < words ? min(32u, c.num_blocks - w * 32) : 0u;
        uint32_t bits = w < words ? c.free_mask[w] : 0u;
        if (in_word < 32) bits &= (1u << in_word) - 1u;
        uint32_t sum;
        const uint32_t before = plan_scan(in_word - static_cast<uint32_t>(__popc(bits)), sm, &sum);
        if (w < words) c.plan.used_before[w] = used + before;
        used += sum;
    }
    if (threadIdx.x == 0) c.plan.used_before[words] = used;
}

// The list of moves: the k-th used page from L on, to the k-th free page.
// forward[id]: where a page goes (its own id where it stays or is free).
__global__ __launch_bounds__(kWideThreads) void pages_moves_kernel(PagesCompact c) {
    const uint32_t words = (c.num_blocks + 31) / 32;
    const uint32_t live = c.plan.used_before[words];
    const uint32_t id = blockIdx.x * kWideThreads + threadIdx.x;
    if (id >= c.num_blocks) return;
    const uint32_t bit = 1u << (id & 31), bits = c.free_mask[id >> 5];
    const uint32_t used_before = c.plan.used_before[id >> 5] + static_cast<uint32_t>(__popc(~bits & (bit - 1)));
    const bool free_page = (bits & bit) != 0;
    if (free_page && id < live) c.plan.to[id - used_before] = static_cast<int32_t>(id);
    if (!free_page && id >= live) {
        // used pages before L: what is used before this one, less its rank among the movers
        const uint32_t lw = live >> 5, below = live < c.num_blocks ? c.plan.used_before[lw] + static_cast<uint32_t>(__popc(~c.free_mask[lw] & ((1u << (live & 31)) - 1u))) : live;
        c.plan.from[used_before - below] = static_cast<int32_t>(id);
        c.plan.rank[id] = static_cast<int32_t>(used_before - below);
    } else {
        c.plan.rank[id] = -1;
    }
    if (id == live || (live == c.num_blocks && id == 0)) {
        const uint32_t below = live == c.num_blocks ? live : used_before;
        *c.plan.moves = live - below;
    }
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
    hipLaunchKernelGGL(pages_fork_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, f);
    const uint32_t groups = f.rows_in + f.rows_out + f.rows_out * planes.layers;
    hipLaunchKernelGGL(pages_fork_kernel, dim3(groups), dim3(kWideThreads), 0, st, f, planes);
    return static_cast<int>(hipGetLastError());
}

int launch_pages_compact(const PagesCompact &c, const PagePlanes &planes, void *stream) {
    const hipStream_t st = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(pages_count_kernel, dim3(1), dim3(kPlanThreads), 0, st, c);
    hipLaunchKernelGGL(pages_moves_kernel, dim3((c.num_blocks + kWideThreads - 1) / kWideThreads), dim3(kWideThreads), 0, st, c);
    const uint64_t copies = static_cast<uint64_t>(c.num_blocks / 2 + 1) * planes.layers, entries = static_cast<uint64_t>(c.rows) * c.max_blocks + c.num_blocks;
    const uint32_t copy_groups = static_cast<uint32_t>(copies < 2048 ? copies : 2048);
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
