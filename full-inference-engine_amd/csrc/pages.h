// Pages of a cache: rows fork, are cut and grown, shared last pages copied, pages moved
// together (fie_pages_*).
#pragma once

#include "copy.h"
#include "fie_decode.h"

namespace fie {

constexpr int kPageBlock = 1024;                        // pages of one count of free ones
constexpr int kPageThreads = 1024;

// The state's parts.
struct PageState {
    int32_t *table, *lengths, *refs, *blocks;
    int pages, page, rows, wide, nblocks;
};

struct PageCopy {
    int32_t src, dst, fill;             // fill: tokens
};

struct PageScratch {
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

// C columns from c0 on, or (C 0) all columns, of all rows' tables go through LDS (`tile`), so that rows may
// take each other's.  A page is in one column of all rows that hold it, so one workgroup sees all
// changes to its count: what is added first, then, behind a barrier, what is taken; a count that
// gets to 0 is a page set free, counted by blocks in LDS (`freed`, [nblocks]).
template <int C, int T>
FIE_DEV void fork_columns(const PageState& s, const int32_t* parents, const int32_t* lengths, int c0,
                          int32_t* tile, int32_t* keep, uint16_t* from, int32_t* freed)
{
    const int tid = threadIdx.x, pitch = C ? C : s.wide;
    auto each = [&](auto&& f) {                         // f(row, column)
        if constexpr (C > 0) {
#pragma unroll 2
            for (int i = tid; i < s.rows * C; i += T) f(i / C, i % C);
        } else {
#pragma unroll 1
            for (int row = tid >> 6; row < s.rows; row += T / 64)
#pragma unroll 1
                for (int c = tid & 63; c < s.wide; c += 64) f(row, c);
        }
    };
    each([&](int row, int c) { tile[row * pitch + c] = c0 + c < s.wide ? s.table[(int64_t)row * s.wide + c0 + c] : -1; });
#pragma unroll 1
    for (int i = tid; i < s.rows; i += T) {
        const int p = page_parent(parents, i, s.rows);
        keep[i] = (int)(((uint32_t)page_held(s, lengths, i, p) + (uint32_t)s.page - 1u) / (uint32_t)s.page);
        from[i] = (uint16_t)(p < 0 ? i : p);            // without a parent nothing is kept
    }
#pragma unroll 1
    for (int i = tid; i < s.nblocks; i += T) freed[i] = 0;
    __syncthreads();
    auto fresh = [&](int row, int c) { return c0 + c < keep[row] ? tile[(int)from[row] * pitch + c] : -1; };
    each([&](int row, int c) {
        const int is = fresh(row, c);
        if (tile[row * pitch + c] == is) return;
        s.table[(int64_t)row * s.wide + c0 + c] = is;
        if (is >= 0) atomicAdd(&s.refs[is], 1);
    });
    __syncthreads();                                    // (a workgroup's own order is enough, and far cheaper than the device's)
    each([&](int row, int c) {
        const int was = tile[row * pitch + c];
        if (was >= 0 && was != fresh(row, c) && atomicAdd(&s.refs[was], -1) == 1) atomicAdd(&freed[was / kPageBlock], 1);
    });
}

// A workgroup C columns of all rows (512 rows of 142 pages 7 us; with fences of the device's scope 14).
// Dynamic LDS: [rows][C] entries, [rows] pages kept, [nblocks],
// [rows] parents.
template <int C>
__global__ __launch_bounds__(kPageThreads) void k_pages_fork(const PageState s, const int32_t* parents, const int32_t* lengths)
{
    extern __shared__ int32_t L[];
    int32_t* const keep = L + s.rows * C;
    int32_t* const freed = keep + s.rows;
    fork_columns<C, kPageThreads>(s, parents, lengths, blockIdx.x * C, L, keep, (uint16_t*)(freed + s.nblocks), freed);
    __syncthreads();
#pragma unroll 1
    for (int b = threadIdx.x; b < s.nblocks; b += kPageThreads)
        if (freed[b]) atomicAdd(&s.blocks[b], freed[b]);
}

// Exclusive prefix sums over the threads of a workgroup of T, sums past 2^30 as 2^30 (a wave's
// own are below 2^31); all the sums.  `part` [T / 64].
constexpr int kScanMost = 1 << 30;
template <int T> FIE_DEV int block_scan(int v, int32_t* part, int* all)
{
    const int wave = threadIdx.x >> 6;
    const int incl = (int)wave_incl_scan_u32((uint32_t)v);
    __syncthreads();                                    // part may still be read from before
    if ((threadIdx.x & 63) == 63) part[wave] = incl;
    __syncthreads();
    int64_t before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < T / 64; ++w) {
        const int t = part[w];
        before += w < wave ? t : 0;
        sum += t;
    }
    *all = (int)min(sum, (int64_t)kScanMost);
    return (int)min(before + incl - v, (int64_t)kScanMost);
}

// Last pages that rows grow from and others hold, by their number: how many rows grow from each, and
// the longest of these, then lowest (`slots` a power of two past 1.5 times the rows).
struct PageMarks {
    int32_t *key, *count;
    uint32_t* best;
    int bits;
    FIE_DEV int slot(int p) const { return (int)(((uint32_t)p * 0x9E3779B1u) >> (32 - bits)); }
    template <int T> FIE_DEV void clear() const
    {
#pragma unroll 1
        for (int i = threadIdx.x; i < 1 << bits; i += T) {
            key[i] = -1;
            count[i] = 0;
            best[i] = 0;
        }
    }
    FIE_DEV void add(int p, uint32_t code) const
    {
        int i = slot(p);
#pragma unroll 1
        for (;; i = (i + 1) & ((1 << bits) - 1)) {
            const int was = atomicCAS(&key[i], -1, p);
            if (was == -1 || was == p) break;
        }
        atomicAdd(&count[i], 1);
        atomicMax(&best[i], code);
    }
    FIE_DEV int find(int p) const
    {
        int i = slot(p);
#pragma unroll 1
        while (key[i] != p) i = (i + 1) & ((1 << bits) - 1);
        return i;
    }
};

// Dynamic LDS of k_pages_grow in ints: held, keep, end [rows], base [nblocks]; then the marks, and in
// their place later the list of free pages (or, with FORK, the table's tile before them).
static inline int mark_bits(int rows)
{
    int b = 4;
    while ((1 << b) < rows + rows / 2) ++b;
    return b;
}

// One workgroup: which rows grow, which last pages are copied, and which pages they get.  The free
// pages are found by the counts of their blocks, so only blocks are read that have some of the
// wanted.  FORK: a small table's rows take their parents' pages first, by the same workgroup (4 x 37: 6 us
// and a launch less).  A chain of dependent steps through memory: parents, lengths, a row's last
// page, its count, the blocks' pages.  512 rows 10 us (marks in memory, unrolled loops: 22), 4 rows with
// their table 8.4 (1024 threads 9.6).
template <bool FORK, int T>
__global__ __launch_bounds__(T) void k_pages_grow(const PageState s, const PageScratch w, const int32_t* parents,
                                                             const int32_t* lengths, uint8_t* granted, int bits, int room)
{
    extern __shared__ int32_t L[];
    __shared__ int32_t part[16];
    __shared__ int32_t copies;
    int32_t* const held = L;
    int32_t* const keep = held + s.rows;
    int32_t* const end = keep + s.rows;
    int32_t* const base = end + s.rows;
    int32_t* const area = base + s.nblocks;
    const PageMarks marks{area, area + (1 << bits), (uint32_t*)(area + (2 << bits)), bits};
    const int tid = threadIdx.x, lane = tid & 63;
    const int each = (s.rows + T - 1) / T, first = tid * each, last = min(first + each, s.rows);
    if (tid == 0) copies = 0;
    if constexpr (FORK) {
        fork_columns<0, T>(s, parents, lengths, 0, area, keep, (uint16_t*)end, base);
        __syncthreads();
    }
    const uint32_t page = (uint32_t)s.page;
    auto wants = [&](int i) { return lengths ? max(lengths[i], held[i]) : held[i]; };
    auto up = [&](int tokens) { return (int)(((uint32_t)tokens + page - 1u) / page); };
    // each thread's rows: what is held, and a last page that is not full, is to be written and that
    // others hold
#pragma unroll 1
    for (int i = first; i < last; ++i) {
        const int h = page_held(s, lengths, i, page_parent(parents, i, s.rows));
        held[i] = h;
        keep[i] = up(h);
    }
    if (lengths) marks.template clear<T>();
    __syncthreads();
#pragma unroll 1
    for (int i = first; i < last; ++i) {
        const int h = held[i], want = wants(i), fill = h - max(keep[i] - 1, 0) * s.page;
        int p = -1;
        if (want > h && up(want) <= s.wide && fill < s.page && h) {
            p = s.table[(int64_t)i * s.wide + keep[i] - 1];
            if (s.refs[p] > 1) marks.add(p, ((uint32_t)fill << 13) | (uint32_t)(s.rows - i));
            else p = -1;
        }
        end[i] = p;
    }
    __syncthreads();
    // what each row wants, a copy in the sign bit
    int mine = 0;
#pragma unroll 1
    for (int i = first; i < last; ++i) {
        const int h = held[i], want = wants(i), fill = h - max(keep[i] - 1, 0) * s.page, p = end[i];
        bool copy = false;
        if (p >= 0) {
            const int m = marks.find(p);
            copy = !(marks.count[m] == s.refs[p] && marks.best[m] == (((uint32_t)fill << 13) | (uint32_t)(s.rows - i)));
        }
        const int demand = want > h && up(want) <= s.wide ? up(want) - keep[i] + copy : 0;
        end[i] = demand | (copy ? (int)0x80000000 : 0);
        mine += demand;
    }
    int sum;
    int at = block_scan<T>(mine, part, &sum);
    // where the free pages of each block begin
    int free = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < s.nblocks; b0 += T) {
        const int b = b0 + tid;
        const int v = b < s.nblocks ? s.blocks[b] + (FORK ? base[b] : 0) : 0;
        const int before = block_scan<T>(v, part, &sum);
        if (b < s.nblocks) base[b] = free + before;
        free += sum;
    }
    int need = 0;                                       // pages that are given out
#pragma unroll 1
    for (int i = first; i < last; ++i) {
        const int demand = end[i] & 0x7FFFFFFF;
        at += demand;
        if (demand && at <= free) need = at;
        end[i] = at | (end[i] & (int)0x80000000);
    }
    need = (int)wave_max_u32((uint32_t)need);
    __syncthreads();
    if (lane == 0) part[tid >> 6] = need;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < T / 64; ++v) need = max(need, part[v]);
    // the first `need` free pages, a wave a block; the blocks' counts without them
    int32_t* const list = need <= room ? area : w.list;
#pragma unroll 1
    for (int b = __builtin_amdgcn_readfirstlane(tid >> 6); b < s.nblocks && base[b] < need; b += T / 64) {
        const int next = b + 1 < s.nblocks ? base[b + 1] : free;
        if (next == base[b]) continue;
        int rank = base[b];
        uint32_t is = 0;                                // bit j: page 64 j + lane is free
#pragma unroll
        for (int j = 0; j < kPageBlock / 64; ++j) is |= (uint32_t)(s.refs[min(b * kPageBlock + j * 64 + lane, s.pages - 1)] == 0) << j;
#pragma unroll 1
        for (int j = 0; j < kPageBlock / 64; ++j) {
            const int p = b * kPageBlock + j * 64 + lane;
            const bool mine = ((is >> j) & 1u) && p < s.pages;
            const uint64_t m = __ballot(mine);
            const int r = rank + (int)__popcll(m & ((1ull << lane) - 1ull));
            if (mine && r < need) list[r] = p;
            rank += (int)__popcll(m);
        }
        if (!FORK && lane == 0) s.blocks[b] = next - min(next, need);
    }
    if constexpr (FORK) {
#pragma unroll 1
        for (int b = tid; b < s.nblocks; b += T) {
            const int next = b + 1 < s.nblocks ? base[b + 1] : free;
            s.blocks[b] = next - max(base[b], min(next, need));
        }
    }
    __syncthreads();
    // a page for each that is wanted: the first row whose sum is past its number has it
#pragma unroll 1
    for (int n = tid; n < need; n += T) {
        int lo = 0, hi = s.rows - 1;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if ((end[mid] & 0x7FFFFFFF) > n) hi = mid;
            else lo = mid + 1;
        }
        const int i = lo, before = i ? end[i - 1] & 0x7FFFFFFF : 0;
        const bool copy = end[i] < 0;
        const int p = list[n];
        int32_t* to = s.table + (int64_t)i * s.wide + keep[i] + (n - before) - copy;    // a copy's first is the last page itself
        if (copy && n == before) {
            const int was = *to;
            atomicAdd(&s.refs[was], -1);                // others hold it
            w.copies[atomicAdd(&copies, 1)] = PageCopy{was, p, held[i] - (keep[i] - 1) * s.page};
        }
        *to = p;
        s.refs[p] = 1;
    }
    __syncthreads();
#pragma unroll 1
    for (int i = first; i < last; ++i) {
        const int want = wants(i), u = up(want);
        const bool grow = want > held[i];
        const bool gets = !grow || (u <= s.wide && ((end[i] & 0x7FFFFFFF) <= free || u - keep[i] + (end[i] < 0) == 0));
        granted[i] = gets;
        s.lengths[i] = grow && gets ? want : held[i];
    }
    if (tid == 0) *w.count = copies;
}

// Moved pages and used pages of a compaction.
struct PageMoves {
    int moved, used;
};

// The block's 1024 pages: free ones below the count of used pages are holes, used ones past it move;
// both are numbered in order.
FIE_DEV PageMoves number_block(const PageState& s, const PageScratch& w, int block, int32_t* part)
{
    const int tid = threadIdx.x;
    int free = 0, before = 0, below = 0;
    for (int b = tid; b < s.nblocks; b += kPageThreads) free += s.blocks[b];
    block_scan<kPageThreads>(free, part, &free);
    const int used = s.pages - free, edge = used / kPageBlock;      // the block that the count falls into
    for (int b = tid; b < s.nblocks; b += kPageThreads) {
        before += b < block ? s.blocks[b] : 0;
        below += b < edge ? s.blocks[b] : 0;
    }
    const int q = edge * kPageBlock + tid;
    below += q < used && s.refs[q] == 0;
    block_scan<kPageThreads>(before, part, &before);
    block_scan<kPageThreads>(below, part, &below);                  // free pages below the count
    const int p = block * kPageBlock + tid;
    const bool in = p < s.pages, is_free = in && s.refs[p] == 0;
    int sum;
    const int rank = before + block_scan<kPageThreads>(is_free, part, &sum);    // of free pages below p
    if (is_free && p < used) w.list[rank] = p;
    if (in && !is_free && p >= used) {
        const int n = (p - rank) - (used - below);                  // used pages below p, less those below the count
        w.movers[n] = p;
        w.order[p] = n;
    }
    return PageMoves{below, used};
}

// Table entries, counts and blocks after the move: every `step`-th from `at` on.
FIE_DEV void rename_pages(const PageState& s, const PageScratch& w, PageMoves m, int64_t at, int64_t step)
{
    const int64_t n = (int64_t)s.rows * s.wide;
    for (int64_t i = at; i < n; i += step) {
        const int p = s.table[i];
        if (p >= m.used) s.table[i] = w.list[w.order[p]];
    }
    for (int64_t i = at; i < m.moved; i += step) {
        s.refs[w.list[i]] = s.refs[w.movers[i]];
        s.refs[w.movers[i]] = 0;
    }
    for (int64_t b = at; b < s.nblocks; b += step) {
        const int size = min(kPageBlock, s.pages - (int)b * kPageBlock);
        s.blocks[b] = max(0, min(size, (int)b * kPageBlock + size - m.used));
    }
}

// A workgroup a block; ALL: one workgroup all of a small pool's, and its table (8 rows: 2 us and a
// launch less).
template <bool ALL>
__global__ __launch_bounds__(kPageThreads) void k_pages_holes(const PageState s, const PageScratch w, int32_t* live)
{
    __shared__ int32_t part[16];
    PageMoves m{0, 0};
    if constexpr (ALL) {
        for (int b = 0; b < s.nblocks; ++b) m = number_block(s, w, b, part);
        __syncthreads();
        rename_pages(s, w, m, threadIdx.x, kPageThreads);
    } else m = number_block(s, w, blockIdx.x, part);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        w.count[0] = m.moved;
        w.count[1] = m.used;
        if (live) *live = m.used;
    }
}

__global__ __launch_bounds__(256) void k_pages_rename(const PageState s, const PageScratch w)
{
    rename_pages(s, w, PageMoves{w.count[0], w.count[1]}, (int64_t)blockIdx.x * 256 + threadIdx.x, (int64_t)gridDim.x * 256);
}

// Where a call's copies stand: k_pages_grow's, lists of two arrays, or the caller's.
struct PageList {
    const PageCopy* copies;
    const int32_t *src, *dst;
    const int32_t* count;           // on the device, or NULL:
    int n, pages;                   // so many
};

// Pieces of pages of one layout: grid (pieces of a page in all caches, copies or fewer).  5400 pages of
// 32 KB in two caches 130 us (5.4 TB/s), 100 pages of 16 KB 3.
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
