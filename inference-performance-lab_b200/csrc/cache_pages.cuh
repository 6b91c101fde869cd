// Pages of a KV cache: claiming, sharing, copying, releasing and compacting them on the device.
//
// State: block tables [rows, width] (entry j of a row is the page of its tokens j * page_size and on,
// -1 where there is none), sequence lengths [rows] and a reference count per page; a page is free
// when its count is 0. Nothing else is kept, so there is no free list to corrupt, and a claim always
// takes the lowest-numbered free pages in order: results do not depend on timing.
#pragma once

#include "ipl_common.cuh"

namespace ipl {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / kWarpSize;
constexpr int kPageCopyThreads = 128;  // a CTA a page
constexpr int kPageMoveThreads = 256;  // CTAs that take pages in turn (377 MB moved: 129 us, with 128 threads 134)
constexpr int kReleaseThreads = 128;
constexpr int kMaxCachesPerLaunch = 128;

// Status of a claim: 0, the number of pages lacking, or this for an argument that is out of range
// (a row, a length, a page, a duplicate row, a child that still holds tokens). Nothing has changed
// unless it is 0.
constexpr int kClaimInvalid = -1;
constexpr int32_t kRowMarked = INT32_MIN;  // sign bit of a length: its row is already in this call

struct PageState {
    int32_t* tables;
    int64_t table_row;
    int32_t* lens;
    int32_t* ref_counts;
    int num_rows, width, num_pages, page_size;
};

struct CacheList {
    char* cache[kMaxCachesPerLaunch];
};

// a + b of non-negative numbers, INT32_MAX where the sum is past it.
__device__ __forceinline__ int saturating_add(int a, int b) {
    return static_cast<int>(min(static_cast<unsigned>(a) + static_cast<unsigned>(b), static_cast<unsigned>(INT32_MAX)));
}

// Exclusive prefix sum of non-negative numbers over the CTA, saturating; `total` gets the sum. `warp_sums`: kPlanWarps ints of shared
// memory, free for reuse after the call's own barriers.
__device__ __forceinline__ int block_exclusive_sum(int value, int* warp_sums, int* total) {
    const int lane = threadIdx.x % kWarpSize, warp = threadIdx.x / kWarpSize;
    int inclusive = value;
#pragma unroll
    for (int offset = 1; offset < kWarpSize; offset *= 2) {
        const int below = __shfl_up_sync(0xffffffffu, inclusive, offset);
        if (lane >= offset) inclusive = saturating_add(inclusive, below);
    }
    if (lane == kWarpSize - 1) warp_sums[warp] = inclusive;
    __syncthreads();
    if (warp == 0) {
        int sum = lane < kPlanWarps ? warp_sums[lane] : 0;
#pragma unroll
        for (int offset = 1; offset < kWarpSize; offset *= 2) {
            const int below = __shfl_up_sync(0xffffffffu, sum, offset);
            if (lane >= offset) sum = saturating_add(sum, below);
        }
        if (lane < kPlanWarps) warp_sums[lane] = sum;
    }
    __syncthreads();
    const int before = warp == 0 ? 0 : warp_sums[warp - 1];
    *total = warp_sums[kPlanWarps - 1];
    __syncthreads();
    return saturating_add(before, inclusive - value);
}

// ---- claiming pages ----------------------------------------------------------------------------

struct ClaimParams {
    PageState state;
    const int32_t* parents;   // fork; null: reserve
    const int32_t* rows;      // fork: the children; reserve: the rows that grow
    const int32_t* new_lens;  // reserve
    int count;                // at most kMaxClaimRows
    int32_t* status;
};
constexpr int kMaxClaimRows = 16384;  // two words of shared memory each
constexpr int kClaimPages = 4;        // pages a thread looks at in a round

__device__ __forceinline__ int pages_of(int len, int page_size) { return len / page_size + (len % page_size != 0); }

// One CTA. Counts the pages each row needs (fork: one where the parent's last page is partly filled) and the
// free ones, and only if they suffice changes anything: the tables' new entries, the counts and the lengths.
// The shared pages and the data of a fork follow in page_fork_kernel.
template <bool kFork>
__global__ void __launch_bounds__(kPlanThreads) page_claim_kernel(const ClaimParams p) {
    extern __shared__ int claim_rows[];
    int* const first = claim_rows;           // rank of a row's first fresh page; -1: not marked by this entry
    int* const base_len = claim_rows + p.count;  // fork: the parent's length; reserve: the row's
    __shared__ int warp_sums[kPlanWarps];
    __shared__ int invalid;
    const PageState& s = p.state;
    const int tid = threadIdx.x;
    if (tid == 0) invalid = 0;
    __syncthreads();
    grid_dependency_wait();
    grid_launch_dependents();

    int needed = 0;
    for (int base = 0; base < p.count; base += kPlanThreads) {
        const int i = base + tid;
        int need = 0;
        bool marked = false;
        if (i < p.count) {
            const int row = p.rows[i];
            bool ok = row >= 0 && row < s.num_rows;
            int len = 0;
            if (ok) {
                // A row that appears twice finds the mark of its first appearance.
                len = atomicOr(&s.lens[row], kRowMarked);
                marked = ok = len >= 0;
            }
            if (kFork) {
                const int parent = p.parents[i];
                int parent_len = 0;
                ok = ok && len == 0 && parent >= 0 && parent < s.num_rows;
                if (ok) {
                    parent_len = *static_cast<volatile int32_t*>(&s.lens[parent]) & ~kRowMarked;
                    ok = pages_of(parent_len, s.page_size) <= s.width;
                }
                base_len[i] = parent_len;
                need = ok && parent_len % s.page_size != 0;
            } else {
                base_len[i] = len;
                if (ok) {
                    const int new_len = p.new_lens[i];
                    ok = new_len >= 0 && pages_of(new_len, s.page_size) <= s.width;
                    if (ok) need = max(0, pages_of(new_len, s.page_size) - pages_of(len, s.page_size));
                }
            }
            if (!ok) invalid = 1;
        }
        int total = 0;
        const int before = block_exclusive_sum(need, warp_sums, &total);
        if (i < p.count) first[i] = marked ? saturating_add(needed, before) : -1;
        needed = saturating_add(needed, total);
    }

    int found = 0;
    for (int base = 0; base < s.num_pages && found < needed; base += kPlanThreads * kClaimPages) {
        int free = 0;
        for (int i = 0; i < kClaimPages; ++i) {
            const int page = base + tid * kClaimPages + i;
            free += page < s.num_pages && s.ref_counts[page] == 0;
        }
        int total = 0;
        block_exclusive_sum(free, warp_sums, &total);
        found += total;
    }
    __syncthreads();
    const int status = invalid ? kClaimInvalid : found < needed ? needed - found : 0;
    if (tid == 0) *p.status = status;
    for (int i = tid; i < p.count; i += kPlanThreads) {
        if (first[i] < 0) continue;
        const int row = p.rows[i];
        s.lens[row] = status != 0 ? (kFork ? s.lens[row] & ~kRowMarked : base_len[i]) : kFork ? base_len[i] : max(base_len[i], p.new_lens[i]);
    }
    if (status != 0) return;
    // The k-th free page goes to the last row whose first rank is at most k.
    found = 0;
    for (int base = 0; found < needed; base += kPlanThreads * kClaimPages) {
        bool is_free[kClaimPages];
        int free = 0;
#pragma unroll
        for (int i = 0; i < kClaimPages; ++i) {
            const int page = base + tid * kClaimPages + i;
            is_free[i] = page < s.num_pages && s.ref_counts[page] == 0;
            free += is_free[i];
        }
        int total = 0;
        int rank = found + block_exclusive_sum(free, warp_sums, &total);
        found += total;
#pragma unroll
        for (int i = 0; i < kClaimPages; ++i) {
            if (!is_free[i] || rank >= needed) continue;
            int lo = 0, hi = p.count - 1;
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (first[mid] <= rank) lo = mid;
                else hi = mid - 1;
            }
            const int page = base + tid * kClaimPages + i;
            const int entry = kFork ? base_len[lo] / s.page_size : pages_of(base_len[lo], s.page_size) + rank - first[lo];
            s.tables[p.rows[lo] * s.table_row + entry] = page;
            s.ref_counts[page] = 1;
            ++rank;
        }
    }
}

// ---- copying pages -----------------------------------------------------------------------------

// `bytes` from one page to another of one cache, by the whole CTA: HBM-bound. 32-byte accesses where pages allow them
// (`wide`), four a thread in flight in copies and forks, two in the compaction; else four of 16 bytes. 96 pages of
// 64 KB in 56 caches, 704 MB read and written: 109 us with CTAs of 128 threads a page, 6.4 TB/s; 111 with two in
// flight, 115 with 16-byte accesses. A compaction of 411 moves in its CTAs of 256 threads: 129 us with two, 137 with
// four.
constexpr int kCopyUnroll = 4, kMoveUnroll = 2;

template <typename Vec, int kUnroll>
__device__ __forceinline__ void copy_vectors(const char* src, char* dst, int64_t bytes) {
    const int64_t step = static_cast<int64_t>(blockDim.x) * sizeof(Vec);
    const auto load = [](const char* p) {
        if constexpr (sizeof(Vec) == 32) return ld_v8(p);
        else return ld_v4(p);
    };
    const auto store = [](char* p, const Vec& v) {
        if constexpr (sizeof(Vec) == 32) st_v8(p, v);
        else st_v4(p, v);
    };
    int64_t at = threadIdx.x * sizeof(Vec);
    for (; at + (kUnroll - 1) * step < bytes; at += kUnroll * step) {
        Vec v[kUnroll];
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) v[i] = load(src + at + i * step);
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) store(dst + at + i * step, v[i]);
    }
    for (; at < bytes; at += step) store(dst + at, load(src + at));
}
struct PageLayout {
    int64_t stride, bytes;  // multiples of 16
    bool wide;              // and of 32, with bases alike
};
template <int kWideUnroll>
__device__ __forceinline__ void copy_page(char* cache, const PageLayout& page, int from, int to) {
    const char* src = cache + from * page.stride;
    char* dst = cache + to * page.stride;
    if (page.wide) copy_vectors<U32x8, kWideUnroll>(src, dst, page.bytes);
    else copy_vectors<U32x4, 4>(src, dst, page.bytes);
}

struct CopyPagesParams {
    CacheList caches;
    int num_caches, count;
    const int32_t* pairs;  // [count, 2]: source, target
    int num_pages;
    PageLayout page;
};

// A CTA for each pair and cache.
__global__ void __launch_bounds__(kPageCopyThreads) page_copy_kernel(const __grid_constant__ CopyPagesParams p) {
    grid_dependency_wait();
    grid_launch_dependents();
    const uint32_t cache = blockIdx.x / p.count, pair = blockIdx.x - cache * p.count;
    const int from = p.pairs[2 * pair], to = p.pairs[2 * pair + 1];
    if (from < 0 || to < 0) return;  // an unused entry
    if (from >= p.num_pages || to >= p.num_pages) {
        if (threadIdx.x == 0) atomicOr(&g_fault_word, kFaultIndexOutOfRange);
        return;
    }
    copy_page<kCopyUnroll>(p.caches.cache[cache], p.page, from, to);
}

struct ForkParams {
    CacheList caches;
    int num_caches, count;
    bool with_tables;  // the first launch of a call that needs several
    PageState state;
    const int32_t* parents;
    const int32_t* children;
    const int32_t* status;
    PageLayout page;
};

// A CTA for each child and cache: the child takes the parent's whole pages (one more reference each)
// and a copy of its partly filled one.
__global__ void __launch_bounds__(kPageCopyThreads) page_fork_kernel(const __grid_constant__ ForkParams p) {
    grid_dependency_wait();
    grid_launch_dependents();
    if (*p.status != 0) return;
    const PageState& s = p.state;
    // Cache after cache, so that a parent's page is read from HBM once for all of its children. Release, fork and
    // reserve of 96 children of 16 parents in 56 caches: 87 us, child after child 121 (with two
    // accesses in flight; with four, cache after cache is still 87). Where the 59 MB of parents'
    // pages are in L2 already, the two orders are level (release and fork 77 and 78 us, 76 since).
    const uint32_t cache = blockIdx.x / p.count, child = blockIdx.x - cache * p.count;
    const int row = p.children[child], len = s.lens[row];  // the parent's
    const int whole = len / s.page_size, used = len % s.page_size;
    const int32_t* from = s.tables + p.parents[child] * s.table_row;
    int32_t* to = s.tables + row * s.table_row;
    if (cache == 0 && p.with_tables) {
        for (int j = threadIdx.x; j < whole; j += kPageCopyThreads) {
            const int page = from[j];
            to[j] = page;
            if (page >= 0 && page < s.num_pages) atomicAdd(&s.ref_counts[page], 1);
            else atomicOr(&g_fault_word, kFaultIndexOutOfRange);
        }
    }
    if (used == 0) return;
    const int last = from[whole];
    if (last < 0 || last >= s.num_pages) {
        if (threadIdx.x == 0) atomicOr(&g_fault_word, kFaultIndexOutOfRange);
        return;
    }
    copy_page<kCopyUnroll>(p.caches.cache[cache], p.page, last, to[whole]);
}

// ---- releasing ---------------------------------------------------------------------------------

// A CTA for each row: every page of the row loses one reference, its entries become -1, its length 0.
// An entry is taken by an exchange, so that a row given twice is released once.
__global__ void __launch_bounds__(kReleaseThreads) page_release_kernel(const PageState s, const int32_t* rows) {
    grid_dependency_wait();
    grid_launch_dependents();
    const int row = rows[blockIdx.x];
    if (row < 0 || row >= s.num_rows) {
        if (threadIdx.x == 0) atomicOr(&g_fault_word, kFaultIndexOutOfRange);
        return;
    }
    // Every entry that holds a page, whatever the length says: it may already be 0 for a row given twice.
    int32_t* table = s.tables + row * s.table_row;
    for (int j = threadIdx.x; j < s.width; j += kReleaseThreads) {
        if (table[j] == -1) continue;
        const int page = atomicExch(&table[j], -1);
        if (page == -1) continue;
        if (page < 0 || page >= s.num_pages || atomicSub(&s.ref_counts[page], 1) <= 0) {
            if (page >= 0 && page < s.num_pages) atomicAdd(&s.ref_counts[page], 1);
            atomicOr(&g_fault_word, kFaultIndexOutOfRange);
        }
    }
    if (threadIdx.x == 0) s.lens[row] = 0;
}

// ---- compacting --------------------------------------------------------------------------------

struct CompactPlanParams {
    const int32_t* ref_counts;
    int32_t* new_ref_counts;
    int num_pages;
    int32_t* live;   // number of pages in use
    int32_t* moves;  // workspace [1]: number of pages that move
    int32_t* map;    // workspace [num_pages]: a page's new number, -1 for a free one
    int32_t* holes;  // workspace [num_pages]
    int32_t* movers;
};

// One CTA: the k-th page in use past the first `live` numbers goes to the k-th free number below.
__global__ void __launch_bounds__(kPlanThreads) page_compact_plan_kernel(const CompactPlanParams p) {
    __shared__ int warp_sums[kPlanWarps];
    grid_dependency_wait();
    grid_launch_dependents();
    const int tid = threadIdx.x;
    int mine = 0;
    for (int page = tid; page < p.num_pages; page += kPlanThreads) mine += p.ref_counts[page] > 0;
    int live = 0;
    block_exclusive_sum(mine, warp_sums, &live);
    int holes = 0, movers = 0;
    for (int base = 0; base < p.num_pages; base += kPlanThreads) {
        const int page = base + tid;
        const int refs = page < p.num_pages ? p.ref_counts[page] : -1;
        const bool hole = page < live && refs <= 0, mover = page >= live && refs > 0;
        int total = 0;
        // Both ranks in one sum: at most 1024 of each a round.
        const int rank = block_exclusive_sum((hole ? 1 : 0) + (mover ? 1 << 16 : 0), warp_sums, &total);
        if (hole) p.holes[holes + (rank & 0xffff)] = page;
        if (mover) p.movers[movers + (rank >> 16)] = page;
        if (page < p.num_pages) {
            p.map[page] = refs > 0 ? page : -1;
            p.new_ref_counts[page] = page < live && refs > 0 ? refs : 0;
        }
        holes += total & 0xffff;
        movers += total >> 16;
    }
    __syncthreads();
    for (int i = tid; i < movers; i += kPlanThreads) {
        const int from = p.movers[i], to = p.holes[i];
        p.map[from] = to;
        p.new_ref_counts[to] = p.ref_counts[from];
    }
    if (tid == 0) {
        *p.live = live;
        *p.moves = movers;
    }
}

struct CompactMoveParams {
    CacheList caches;
    int num_caches;
    const int32_t* tables;  // null in the later launches of a call that needs several
    int32_t* new_tables;
    int64_t table_row;
    int num_rows, width, num_pages;
    const int32_t* moves;
    const int32_t* map;
    const int32_t* holes;
    const int32_t* movers;
    PageLayout page;
};

// Renumbers the tables and moves the pages, a CTA for each page and cache in turn.
__global__ void __launch_bounds__(kPageMoveThreads) page_compact_move_kernel(const __grid_constant__ CompactMoveParams p) {
    grid_dependency_wait();
    grid_launch_dependents();
    if (p.tables != nullptr) {
        const int64_t entries = static_cast<int64_t>(p.num_rows) * p.width;
        for (int64_t e = int64_t{blockIdx.x} * kPageMoveThreads + threadIdx.x; e < entries;
             e += int64_t{gridDim.x} * kPageMoveThreads) {
            const int64_t row = e / p.width, column = e - row * p.width;
            const int page = p.tables[row * p.table_row + column];
            const bool known = page >= 0 && page < p.num_pages;
            p.new_tables[e] = known ? p.map[page] : page;
        }
    }
    const int64_t units = static_cast<int64_t>(*p.moves) * p.num_caches;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int64_t move = u / p.num_caches;
        copy_page<kMoveUnroll>(p.caches.cache[u - move * p.num_caches], p.page, p.movers[move], p.holes[move]);
    }
}

}  // namespace ipl
