// Pages of a cache: rows fork, are cut and grown, shared last pages copied, pages moved
// together (fie_pages_*).
#pragma once

#include "copy.h"
#include "fie_decode.h"

namespace fie {

constexpr int kPageBlock = 1024;                        // pages of one count of free ones
constexpr int kForkThreads = 1024, kForkCols = 8;
constexpr int kGrowThreads = 1024;

// The state's parts.
struct PageState {
    int32_t *table, *lengths, *refs, *blocks;
    int pages, page, rows, wide, nblocks;
};

struct PageCopy {
    int32_t src, dst, fill;             // fill: tokens
};

// The scratch's: `mark` and `writers` are 0 between calls.
struct PageScratch {
    uint64_t* mark;             // [pages] a last page's longest writer, then lowest
    int32_t* writers;           // [pages] rows that grow from it
    int32_t* list;              // [pages] free pages in order; compacting: holes
    int32_t* movers;            // [pages] compacting: used pages past the count, and
    int32_t* order;             // [pages] their numbers among those
    PageCopy* copies;           // [rows]
    int32_t* count;             // [2] copies of this call; compacting: moved pages, used pages
};

FIE_DEV int page_parent(const int32_t* parents, int i, int rows)
{
    const int p = parents ? parents[i] : i;
    return p >= 0 && p < rows ? p : -1;
}

// Tokens that row i keeps of its parent's.
FIE_DEV int page_held(const PageState& s, const int32_t* lengths, int i, int parent)
{
    const int have = parent < 0 ? 0 : s.lengths[parent];
    return lengths ? max(0, min(lengths[i], have)) : have;
}

// A workgroup kForkCols columns of all rows: its table entries go through LDS, so that rows may
// take each other's.  A page is in one column of all rows that hold it, so one workgroup sees all
// changes to its count: what is added first, then, behind a barrier, what is taken; a count
// that gets to 0 is a page set free.  Dynamic LDS: [rows][kForkCols] entries, [rows] pages kept,
// [rows] parents.
__global__ __launch_bounds__(kForkThreads) void k_pages_fork(const PageState s, const int32_t* parents, const int32_t* lengths)
{
    extern __shared__ int32_t L[];
    int32_t* const tile = L;
    int32_t* const keep = L + s.rows * kForkCols;
    uint16_t* const from = (uint16_t*)(keep + s.rows);
    const int tid = threadIdx.x, c0 = blockIdx.x * kForkCols, n = s.rows * kForkCols;
    for (int i = tid; i < n; i += kForkThreads) {
        const int c = c0 + i % kForkCols;
        tile[i] = c < s.wide ? s.table[(int64_t)(i / kForkCols) * s.wide + c] : -1;
    }
    for (int i = tid; i < s.rows; i += kForkThreads) {
        const int p = page_parent(parents, i, s.rows);
        const int held = page_held(s, lengths, i, p);
        keep[i] = (int)(((int64_t)held + s.page - 1) / s.page);
        from[i] = (uint16_t)(p < 0 ? i : p);            // without a parent nothing is kept
    }
    __syncthreads();
    auto fresh = [&](int i) {
        const int row = i / kForkCols, c = i % kForkCols;
        return c0 + c < keep[row] ? tile[(int)from[row] * kForkCols + c] : -1;
    };
    for (int i = tid; i < n; i += kForkThreads) {
        const int was = tile[i], is = fresh(i);
        if (was == is) continue;
        s.table[(int64_t)(i / kForkCols) * s.wide + c0 + i % kForkCols] = is;
        if (is >= 0) atomicAdd(&s.refs[is], 1);
    }
    __threadfence();
    __syncthreads();
    for (int i = tid; i < n; i += kForkThreads) {
        const int was = tile[i];
        if (was == fresh(i) || was < 0) continue;
        if (atomicAdd(&s.refs[was], -1) == 1) atomicAdd(&s.blocks[was / kPageBlock], 1);
    }
}

FIE_DEV int32_t fresh_load(const int32_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
FIE_DEV uint64_t fresh_load(const uint64_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// Exclusive prefix sum over the threads of a workgroup of 1024, sums past 2^30 as 2^30 (a wave's
// own are below 2^31); *total the sum.  `part` [16].
constexpr int kScanMost = 1 << 30;
FIE_DEV int block_scan(int v, int32_t* part, int* total)
{
    const int wave = threadIdx.x >> 6;
    const int incl = (int)wave_incl_scan_u32((uint32_t)v);
    __syncthreads();                                    // part may still be read from before
    if ((threadIdx.x & 63) == 63) part[wave] = incl;
    __syncthreads();
    int64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
        const int t = part[w];
        before += w < wave ? t : 0;
        all += t;
    }
    *total = (int)min(all, (int64_t)kScanMost);
    return (int)min(before + incl - v, (int64_t)kScanMost);
}

// One workgroup: which rows grow, which last pages are copied, and which pages they get.  The free
// pages are found by the counts of their blocks, so only blocks are read that have some of the
// wanted.  Dynamic LDS: [rows] tokens held, [rows] pages wanted up to and with a row, [nblocks].
__global__ __launch_bounds__(kGrowThreads) void k_pages_grow(const PageState s, const PageScratch w, const int32_t* parents,
                                                             const int32_t* lengths, uint8_t* granted)
{
    extern __shared__ int32_t L[];
    __shared__ int32_t part[16];
    __shared__ int32_t copies;
    int32_t* const held = L;
    int32_t* const end = held + s.rows;
    int32_t* const base = end + s.rows;
    const int tid = threadIdx.x;
    const int each = (s.rows + kGrowThreads - 1) / kGrowThreads, first = tid * each, last = min(first + each, s.rows);
    if (tid == 0) copies = 0;
    for (int i = tid; i < s.rows; i += kGrowThreads) held[i] = page_held(s, lengths, i, page_parent(parents, i, s.rows));
    __syncthreads();
    auto wants = [&](int i) { return lengths ? max(lengths[i], held[i]) : held[i]; };
    auto fits = [&](int want) { return (int64_t)want <= (int64_t)s.wide * s.page; };
    auto up = [&](int tokens) { return (int)(((int64_t)tokens + s.page - 1) / s.page); };
    auto part_page = [&](int i, int want) {             // a last page that is not full and is to be written
        return want > held[i] && fits(want) && held[i] % s.page ? s.table[(int64_t)i * s.wide + held[i] / s.page] : -1;
    };
    auto key_of = [&](int i) { return ((uint64_t)(uint32_t)(held[i] % s.page) << 32) | (uint32_t)(s.rows - i); };
    for (int i = first; i < last; ++i) {
        const int p = part_page(i, wants(i));
        if (p >= 0) {
            atomicAdd(&w.writers[p], 1);
            atomicMax((unsigned long long*)&w.mark[p], (unsigned long long)key_of(i));
        }
    }
    __threadfence();
    __syncthreads();
    // what each row wants; end[] holds its sign bit for a copy until the rows' sums are there
    int mine = 0;
    for (int i = first; i < last; ++i) {
        const int want = wants(i), p = part_page(i, want);
        const bool copy = p >= 0 && !(fresh_load(&w.writers[p]) == fresh_load(&s.refs[p]) && fresh_load(&w.mark[p]) == key_of(i));
        const int demand = want > held[i] && fits(want) ? up(want) - up(held[i]) + copy : 0;
        end[i] = demand | (copy ? (int)0x80000000 : 0);
        mine += demand;
    }
    int all;
    int at = block_scan(mine, part, &all);
    // where the free pages of each block begin
    int free = 0;
    for (int b0 = 0; b0 < s.nblocks; b0 += kGrowThreads) {
        const int b = b0 + tid;
        const int v = b < s.nblocks ? fresh_load(&s.blocks[b]) : 0;
        int sum;
        const int before = block_scan(v, part, &sum);
        if (b < s.nblocks) base[b] = free + before;
        free += sum;
    }
    int need = 0;                                       // pages that are given out
    for (int i = first; i < last; ++i) {
        const int demand = end[i] & 0x7FFFFFFF;
        at += demand;
        if (demand && at <= free) need = at;
        end[i] = at | (end[i] & (int)0x80000000);
    }
    for (int d = 32; d; d >>= 1) need = max(need, __shfl_xor(need, d, 64));
    __syncthreads();
    if ((tid & 63) == 0) part[tid >> 6] = need;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < 16; ++v) need = max(need, part[v]);
    // the first `need` free pages, a wave a block
    const int lane = tid & 63;
    for (int b = __builtin_amdgcn_readfirstlane(tid >> 6); b < s.nblocks && base[b] < need; b += kGrowThreads / 64) {
        const int next = b + 1 < s.nblocks ? base[b + 1] : free;
        if (next == base[b]) continue;
        int rank = base[b];
        uint32_t is = 0;                                // bit j: page 64 j + lane is free
#pragma unroll
        for (int j = 0; j < kPageBlock / 64; ++j) {
            const int p = b * kPageBlock + j * 64 + lane;
            if (p < s.pages && fresh_load(&s.refs[p]) == 0) is |= 1u << j;
        }
#pragma unroll
        for (int j = 0; j < kPageBlock / 64; ++j) {
            const uint64_t m = __ballot((is >> j) & 1u);
            const int r = rank + (int)__popcll(m & ((1ull << lane) - 1ull));
            if (((is >> j) & 1u) && r < need) w.list[r] = b * kPageBlock + j * 64 + lane;
            rank += (int)__popcll(m);
        }
    }
    __syncthreads();
    // a page for each that is wanted: the first row whose sum is past its number has it
    for (int n = tid; n < need; n += kGrowThreads) {
        int lo = 0, hi = s.rows - 1;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if ((end[mid] & 0x7FFFFFFF) > n) hi = mid;
            else lo = mid + 1;
        }
        const int i = lo, before = i ? end[i - 1] & 0x7FFFFFFF : 0;
        const bool copy = end[i] < 0;
        const int col = up(held[i]) + (n - before) - copy, p = w.list[n];
        int32_t* to = s.table + (int64_t)i * s.wide + col;      // with a copy, the first is the last page itself
        if (copy && n == before) {
            const int was = *to;
            atomicAdd(&s.refs[was], -1);                        // others hold it
            w.copies[atomicAdd(&copies, 1)] = PageCopy{was, p, held[i] % s.page};
        }
        *to = p;
        s.refs[p] = 1;
        atomicAdd(&s.blocks[p / kPageBlock], -1);
    }
    __syncthreads();
    // the marks go back to 0, the lengths out
    for (int i = first; i < last; ++i) {
        const int want = wants(i), sum = end[i] & 0x7FFFFFFF;
        const bool copy = end[i] < 0, grow = want > held[i], fit = fits(want);
        const bool gets = !grow || (fit && (sum <= free || up(want) - up(held[i]) + copy == 0));
        if (grow && fit && held[i] % s.page && !(copy && gets)) {   // of a copied page the list has its number
            const int p = s.table[(int64_t)i * s.wide + held[i] / s.page];
            w.writers[p] = 0;
            w.mark[p] = 0;
        }
        granted[i] = gets;
        s.lengths[i] = grow && gets ? want : held[i];
    }
    for (int n = tid; n < copies; n += kGrowThreads) {
        w.writers[w.copies[n].src] = 0;
        w.mark[w.copies[n].src] = 0;
    }
    if (tid == 0) *w.count = copies;
}

// A workgroup 1024 pages: free ones below the count of used pages are holes, used ones past it
// move; both are numbered in order.
__global__ __launch_bounds__(kGrowThreads) void k_pages_holes(const PageState s, const PageScratch w, int32_t* live)
{
    __shared__ int32_t part[16];
    const int tid = threadIdx.x, block = blockIdx.x;
    int free = 0, before = 0;
    for (int b = tid; b < s.nblocks; b += kGrowThreads) free += s.blocks[b];
    block_scan(free, part, &free);
    const int used = s.pages - free, edge = used / kPageBlock;      // the block that the count falls into
    int below = 0;
    for (int b = tid; b < s.nblocks; b += kGrowThreads) {
        before += b < block ? s.blocks[b] : 0;
        below += b < edge ? s.blocks[b] : 0;
    }
    const int q = edge * kPageBlock + tid;
    below += q < used && s.refs[q] == 0;
    block_scan(before, part, &before);
    block_scan(below, part, &below);                                // free pages below the count
    const int p = block * kPageBlock + tid;
    const bool in = p < s.pages, is_free = in && s.refs[p] == 0;
    int sum;
    const int rank = before + block_scan(is_free, part, &sum);     // of free pages below p
    if (is_free && p < used) w.list[rank] = p;
    if (in && !is_free && p >= used) {
        const int n = (p - rank) - (used - below);                  // used pages below p, less those below the count
        w.movers[n] = p;
        w.order[p] = n;
    }
    if (block == 0 && tid == 0) {
        w.count[0] = below;
        w.count[1] = used;
        if (live) *live = used;
    }
}

// Table entries, counts and blocks after the move.
__global__ __launch_bounds__(256) void k_pages_rename(const PageState s, const PageScratch w)
{
    const int moved = w.count[0], used = w.count[1];
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, n = (int64_t)s.rows * s.wide, step = (int64_t)gridDim.x * 256;
    for (int64_t i = at; i < n; i += step) {
        const int p = s.table[i];
        if (p >= used) s.table[i] = w.list[w.order[p]];
    }
    for (int64_t i = at; i < moved; i += step) {
        s.refs[w.list[i]] = s.refs[w.movers[i]];
        s.refs[w.movers[i]] = 0;
    }
    for (int64_t b = at; b < s.nblocks; b += step) {
        const int size = min(kPageBlock, s.pages - (int)b * kPageBlock);
        s.blocks[b] = max(0, min(size, (int)(b + 1) * kPageBlock - used - (kPageBlock - size)));
    }
}

// Where a call's copies stand: k_pages_grow's, lists of two arrays, or the caller's.
struct PageList {
    const PageCopy* copies;
    const int32_t *src, *dst;
    const int32_t* count;           // on the device, or NULL:
    int n, pages;                   // so many
};

// Pieces of pages of one layout: grid (pieces of a page in all caches, copies or fewer).
__global__ __launch_bounds__(kCopyThreads) void k_pages_copy(const PageList l, const fie_cache_group g, int page, int chunks)
{
    const int n = l.count ? *l.count : l.n;
    const int per = g.outer * chunks;
    const int c = blockIdx.x / per, unit = blockIdx.x - c * per, piece = unit / chunks, chunk = unit - piece * chunks;
    uint8_t* const base = (uint8_t*)g.base[c] + piece * g.outer_stride;
    for (int i = blockIdx.y; i < n; i += gridDim.y) {
        const PageCopy p = l.copies ? l.copies[i] : PageCopy{l.src[i], l.dst[i], page};
        if ((uint32_t)p.src >= (uint32_t)l.pages || (uint32_t)p.dst >= (uint32_t)l.pages || p.src == p.dst) continue;
        copy_chunk(base + p.dst * g.page_stride, base + p.src * g.page_stride, g.whole ? g.token_bytes : p.fill * g.token_bytes, chunk);
    }
}

}  // namespace fie
