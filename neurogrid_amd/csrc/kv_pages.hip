// kv_pages.hip - the page table of a key/value cache: handing out, sharing,
// giving back and moving together pages (kv_cache.h).
//
// All on the device, so that a decoding step with its page management can be
// captured into a graph. Every result is determined by the inputs: free pages
// are ranked by their number, and reference counts change by atomic additions
// only, whose order does not matter. A launch either reads the counts or changes
// them: a plan first, its effects in a second launch.
#include "kv_cache.hpp"

#include <algorithm>

namespace ng {
namespace {

constexpr int kPgThreads = 1024;
constexpr int kPgMaxRows = 8192;

struct PoolView {
    int* table;
    int* refs;
    int rows, cols, pages, ps_log2;
};

// Sum over the block, in every thread; s holds a value per wave.
template <typename N>
__device__ __forceinline__ N block_sum(N v, N* s) {
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) v += __shfl_xor(v, off, kWave);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < kPgThreads / kWave; ++w) v += s[w];
    __syncthreads();
    return v;
}

// Sum of v over the threads before this one; of all of them in *total.
__device__ __forceinline__ int block_before(int v, int* s, int* total) {
    const int lane = threadIdx.x & 63;
    int x = v;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        const int o = __shfl_up(x, off, kWave);
        if (lane >= off) x += o;
    }
    if (lane == 63) s[threadIdx.x >> 6] = x;
    __syncthreads();
    int before = x - v, sum = 0;
#pragma unroll
    for (int w = 0; w < kPgThreads / kWave; ++w) {
        if (w < static_cast<int>(threadIdx.x >> 6)) before += s[w];
        sum += s[w];
    }
    __syncthreads();
    *total = sum;
    return before;
}

// How many pages of [0, end) are used, and how many of [0, part), part <= end:
// every block counts for itself (the counts stay in L2), 16 loads a thread on
// their way at a time.
__device__ __forceinline__ int used_before(const int* refs, int end, int part, unsigned long long* s, int* in_part) {
    unsigned long long n = 0;  // both counts, end <= 2^30
    for (int i0 = threadIdx.x; i0 < end; i0 += 16 * kPgThreads) {
        int r[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) r[k] = refs[min(i0 + k * kPgThreads, end - 1)];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const int i = i0 + k * kPgThreads;
            if (i < end && r[k] > 0) n += 1ull + (i < part ? 1ull << 32 : 0);
        }
    }
    n = block_sum(n, s);
    *in_part = static_cast<int>(n >> 32);
    return static_cast<int>(n & 0xffffffffull);
}

__device__ __forceinline__ int pages_of(int tokens, int ps_log2) {
    return static_cast<int>((static_cast<uint32_t>(max(tokens, 0)) + (1u << ps_log2) - 1) >> ps_log2);
}

// What row r asks for: entries [have, want) and, if shared, a copy of entry have - 1.
struct Growth {
    int have, want, shared, missing;
};
__device__ __forceinline__ Growth growth(const PoolView& p, const int* old_lens, const int* new_lens, int r) {
    const int o = max(old_lens[r], 0), n = new_lens[r];
    Growth g{0, 0, -1, 0};
    if (n <= o) return g;
    g.have = pages_of(o, p.ps_log2);
    g.want = pages_of(n, p.ps_log2);
    g.missing = max(g.want - p.cols, 0);
    g.want = min(g.want, p.cols);
    g.have = min(g.have, g.want);
    if ((o & ((1 << p.ps_log2) - 1)) != 0 && g.have > 0) {
        const int page = p.table[static_cast<size_t>(r) * p.cols + g.have - 1];
        if (page >= 0 && page < p.pages && p.refs[page] > 1) g.shared = page;
    }
    return g;
}

// Plan: free pages into copy_dst and the new entries of the table. Block i
// looks after the pages from 1024 i on: it counts the free ones before them
// and hands out its own by rank. Every block sums up the rows' needs (first in
// LDS: the rank at which a row's pages start).
__global__ __launch_bounds__(kPgThreads) void kv_grow_plan_kernel(PoolView p, const int* old_lens, const int* new_lens,
                                                                  int* copy_src, int* copy_dst, int* d_missing) {
    __shared__ int first[kPgMaxRows];
    __shared__ int s[kPgThreads / kWave];
    __shared__ unsigned long long s_long[kPgThreads / kWave];
    const int base = blockIdx.x * kPgThreads;
    int need = 0;
    unsigned long long over = 0;
    for (int r0 = 0; r0 < p.rows; r0 += kPgThreads) {
        const int r = r0 + threadIdx.x;
        const Growth g = r < p.rows ? growth(p, old_lens, new_lens, r) : Growth{0, 0, -1, 0};
        int sum;
        const int before = block_before(g.want - g.have + (g.shared >= 0), s, &sum);
        if (r < p.rows) first[r] = need + before;
        need += sum;
        over += static_cast<unsigned>(g.missing);
    }
    over = block_sum(over, s_long);
    int here;
    const int free_all = p.pages - used_before(p.refs, p.pages, base, s_long, &here);
    const int missing = static_cast<int>(min(over + max(need - free_all, 0), 0x7fffffffull));
    if (blockIdx.x == 0) {
        if (threadIdx.x == 0) *d_missing = missing;
        for (int r = threadIdx.x; r < p.rows; r += kPgThreads) {
            const Growth g = growth(p, old_lens, new_lens, r);
            const bool copies = missing == 0 && g.shared >= 0;
            copy_src[r] = copies ? g.shared : -1;
            if (!copies) copy_dst[r] = -1;
        }
    }
    if (missing != 0 || need == 0) return;
    const int free_before = base - here;
    if (free_before >= need) return;
    const int page = base + threadIdx.x;
    const bool is_free = page < p.pages && p.refs[page] <= 0;
    int sum;
    const int rank = free_before + block_before(is_free, s, &sum);
    if (!is_free || rank >= need) return;
    int lo = 0, hi = p.rows - 1;  // the last row that starts at or before rank (rows that need nothing start with their successor)
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= rank) lo = mid; else hi = mid - 1;
    }
    const Growth g = growth(p, old_lens, new_lens, lo);
    int k = rank - first[lo];
    if (g.shared >= 0 && k-- == 0) copy_dst[lo] = page;
    else p.table[static_cast<size_t>(lo) * p.cols + g.have + k] = page;
}

// Effects: counts of the pages given out, and the copied pages' entries.
__global__ __launch_bounds__(256) void kv_grow_apply_kernel(PoolView p, const int* old_lens, const int* new_lens,
                                                            const int* copy_src, const int* copy_dst,
                                                            const int* d_missing) {
    if (*d_missing != 0) return;
    const int r = blockIdx.x, o = max(old_lens[r], 0);
    if (new_lens[r] <= o) return;
    const int have = pages_of(o, p.ps_log2), want = min(pages_of(new_lens[r], p.ps_log2), p.cols);
    for (int i = have + threadIdx.x; i < want; i += 256) {
        const int e = p.table[static_cast<size_t>(r) * p.cols + i];
        if (e >= 0 && e < p.pages) p.refs[e] = 1;
    }
    if (threadIdx.x == 0 && copy_src[r] >= 0) {
        p.refs[copy_dst[r]] = 1;
        atomicSub(&p.refs[copy_src[r]], 1);
        p.table[static_cast<size_t>(r) * p.cols + have - 1] = copy_dst[r];
    }
}

// Row r of the new table, and both tables' changes to the counts: +1 for every
// entry of the new row, -1 for every entry of the old row r.
__global__ __launch_bounds__(256) void kv_fork_kernel(PoolView p, int* new_table, const int* parents, const int* lens,
                                                      int* new_lens) {
    const int r = blockIdx.x, from = parents[r];
    const bool some = from >= 0 && from < p.rows;
    const int n = some ? min(pages_of(lens[from], p.ps_log2), p.cols) : 0;
    const int o = min(pages_of(lens[r], p.ps_log2), p.cols);
    for (int i = threadIdx.x; i < p.cols; i += 256) {
        const int e = i < n ? p.table[static_cast<size_t>(from) * p.cols + i] : -1;
        new_table[static_cast<size_t>(r) * p.cols + i] = e;
        if (e >= 0 && e < p.pages) atomicAdd(&p.refs[e], 1);
        const int was = i < o ? p.table[static_cast<size_t>(r) * p.cols + i] : -1;
        if (was >= 0 && was < p.pages) atomicSub(&p.refs[was], 1);
    }
    if (threadIdx.x == 0) new_lens[r] = some ? max(lens[from], 0) : 0;
}

__global__ __launch_bounds__(256) void kv_free_kernel(PoolView p, const int* old_lens, const int* keep_lens) {
    const int r = blockIdx.x;
    const int keep = pages_of(keep_lens[r], p.ps_log2), o = min(pages_of(old_lens[r], p.ps_log2), p.cols);
    for (int i = keep + threadIdx.x; i < o; i += 256) {
        const size_t at = static_cast<size_t>(r) * p.cols + i;
        const int e = p.table[at];
        p.table[at] = -1;
        if (e >= 0 && e < p.pages) atomicSub(&p.refs[e], 1);
    }
}

// Plan of a compaction: block i ranks the pages from 1024 i on.
__global__ __launch_bounds__(kPgThreads) void kv_compact_plan_kernel(PoolView p, int* copy_src, int* copy_dst,
                                                                     int capacity, int* d_moves) {
    __shared__ int s[kPgThreads / kWave];
    __shared__ unsigned long long s_long[kPgThreads / kWave];
    const int base = blockIdx.x * kPgThreads;
    int here, front, sum;
    const int n = used_before(p.refs, p.pages, base, s_long, &here);
    used_before(p.refs, n, n, s_long, &front);  // used pages before n
    const int moves = n - front;
    const int page = base + threadIdx.x;
    const bool used = page < p.pages && p.refs[page] > 0;
    const int before = here + block_before(used, s, &sum);
    if (page < p.pages) {
        if (used && page >= n) copy_src[before - front] = page;
        if (!used && page < n) copy_dst[page - before] = page;
    }
    for (int k = base + threadIdx.x; k < capacity; k += gridDim.x * kPgThreads)
        if (k >= moves) copy_src[k] = copy_dst[k] = -1;
    if (page == 0) *d_moves = moves;
}

// Its effects: counts move with their pages, entries of the table follow.
__global__ __launch_bounds__(256) void kv_compact_apply_kernel(PoolView p, const int* copy_src, const int* copy_dst,
                                                               const int* d_moves) {
    const int moves = *d_moves;
    const size_t stride = static_cast<size_t>(gridDim.x) * 256, t0 = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
    for (size_t k = t0; k < static_cast<size_t>(moves); k += stride) {
        p.refs[copy_dst[k]] = p.refs[copy_src[k]];
        p.refs[copy_src[k]] = 0;
    }
    if (moves == 0) return;
    const int lowest = copy_src[0];
    const size_t entries = static_cast<size_t>(p.rows) * p.cols;
    for (size_t i = t0; i < entries; i += stride) {
        const int e = p.table[i];
        if (e < lowest) continue;
        int lo = 0, hi = moves - 1;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (copy_src[mid] < e) lo = mid + 1; else hi = mid;
        }
        if (copy_src[lo] == e) p.table[i] = copy_dst[lo];
    }
}

int check_pool(const char* name, const ng_kv_pages* p) {
    NG_REQUIRE(p && p->table && p->refs, "%s: null pointer", name);
    NG_REQUIRE(p->max_seqs > 0 && p->max_pages > 0 && p->num_pages > 0,
               "%s: invalid pool (max_seqs=%d, max_pages=%d, num_pages=%d)", name, p->max_seqs, p->max_pages, p->num_pages);
    NG_REQUIRE(kv_page_ok(p->page_size), "%s: page_size %d is not 16, 32, 64 or 128", name, p->page_size);
    NG_REQUIRE(p->max_pages <= (1 << 30) / p->page_size && p->num_pages <= (1 << 30) &&
                   static_cast<size_t>(p->max_seqs) * p->max_pages <= (size_t(1) << 30) && p->max_seqs <= (1 << 22),
               "%s: the pool is too large", name);
    return 0;
}

PoolView pool_view(const ng_kv_pages& p) {
    return PoolView{static_cast<int*>(p.table), static_cast<int*>(p.refs), p.max_seqs, p.max_pages, p.num_pages,
                    kv_log2(p.page_size)};
}

int page_blocks(int pages) { return (pages + kPgThreads - 1) / kPgThreads; }

}  // namespace
}  // namespace ng

using namespace ng;

extern "C" int ng_kv_pages_grow(const ng_kv_pages* pages, const void* old_lens, const void* new_lens, void* copy_src,
                                void* copy_dst, void* d_missing) {
    const char* name = "ng_kv_pages_grow";
    if (check_pool(name, pages) != 0) return -1;
    NG_REQUIRE(old_lens && new_lens && copy_src && copy_dst && d_missing, "%s: null pointer", name);
    NG_REQUIRE(pages->max_seqs <= kPgMaxRows, "%s: %d sequences are more than %d", name, pages->max_seqs, kPgMaxRows);
    const int* o = static_cast<const int*>(old_lens);
    const int* n = static_cast<const int*>(new_lens);
    int *cs = static_cast<int*>(copy_src), *cd = static_cast<int*>(copy_dst), *miss = static_cast<int*>(d_missing);
    const PoolView p = pool_view(*pages);
    kv_grow_plan_kernel<<<dim3(page_blocks(p.pages)), dim3(kPgThreads), 0, stream()>>>(p, o, n, cs, cd, miss);
    NG_CHECK_LAUNCH(name);
    kv_grow_apply_kernel<<<dim3(p.rows), dim3(256), 0, stream()>>>(p, o, n, cs, cd, miss);
    NG_CHECK_LAUNCH(name);
    return 0;
}

extern "C" int ng_kv_pages_fork(const ng_kv_pages* pages, void* new_table, const void* parents, const void* lens,
                                void* new_lens) {
    const char* name = "ng_kv_pages_fork";
    if (check_pool(name, pages) != 0) return -1;
    NG_REQUIRE(new_table && parents && lens && new_lens, "%s: null pointer", name);
    const size_t bytes = static_cast<size_t>(pages->max_seqs) * pages->max_pages * sizeof(int);
    const auto apart = [](const void* a, const void* b, size_t n) {
        const char *x = static_cast<const char*>(a), *y = static_cast<const char*>(b);
        return x + n <= y || y + n <= x;
    };
    NG_REQUIRE(apart(new_table, pages->table, bytes), "%s: new_table overlaps the table", name);
    NG_REQUIRE(apart(new_lens, lens, pages->max_seqs * sizeof(int)), "%s: new_lens overlaps lens", name);
    kv_fork_kernel<<<dim3(pages->max_seqs), dim3(256), 0, stream()>>>(
        pool_view(*pages), static_cast<int*>(new_table), static_cast<const int*>(parents),
        static_cast<const int*>(lens), static_cast<int*>(new_lens));
    NG_CHECK_LAUNCH(name);
    return 0;
}

extern "C" int ng_kv_pages_free(const ng_kv_pages* pages, const void* old_lens, const void* keep_lens) {
    const char* name = "ng_kv_pages_free";
    if (check_pool(name, pages) != 0) return -1;
    NG_REQUIRE(old_lens && keep_lens, "%s: null pointer", name);
    kv_free_kernel<<<dim3(pages->max_seqs), dim3(256), 0, stream()>>>(
        pool_view(*pages), static_cast<const int*>(old_lens), static_cast<const int*>(keep_lens));
    NG_CHECK_LAUNCH(name);
    return 0;
}

extern "C" int ng_kv_pages_compact(const ng_kv_pages* pages, void* copy_src, void* copy_dst, int capacity,
                                   void* d_moves) {
    const char* name = "ng_kv_pages_compact";
    if (check_pool(name, pages) != 0) return -1;
    NG_REQUIRE(copy_src && copy_dst && d_moves, "%s: null pointer", name);
    NG_REQUIRE(capacity >= pages->num_pages / 2 && capacity > 0, "%s: capacity %d is below num_pages / 2 = %d", name,
               capacity, pages->num_pages / 2);
    NG_REQUIRE(capacity <= (1 << 30), "%s: capacity %d is above 2^30", name, capacity);
    const PoolView p = pool_view(*pages);
    int *cs = static_cast<int*>(copy_src), *cd = static_cast<int*>(copy_dst), *mv = static_cast<int*>(d_moves);
    kv_compact_plan_kernel<<<dim3(page_blocks(p.pages)), dim3(kPgThreads), 0, stream()>>>(p, cs, cd, capacity, mv);
    NG_CHECK_LAUNCH(name);
    const size_t entries = static_cast<size_t>(p.rows) * p.cols;
    const int blocks = static_cast<int>(std::min<size_t>((entries + 255) / 256, 2048));
    kv_compact_apply_kernel<<<dim3(blocks), dim3(256), 0, stream()>>>(p, cs, cd, mv);
    NG_CHECK_LAUNCH(name);
    return 0;
}
