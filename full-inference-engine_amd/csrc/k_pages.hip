// Pages of a cache behind the C ABI of include/fie_decode.h.
#include <algorithm>

#include "launchers.h"
#include "pages.h"

namespace fie {

static PageState page_state(const fie_pages_args& a)
{
    PageState s;
    s.pages = a.pages;
    s.page = a.page;
    s.rows = a.rows;
    s.wide = a.wide;
    s.nblocks = (a.pages + kPageBlock - 1) / kPageBlock;
    s.table = a.state;
    s.lengths = s.table + (int64_t)a.rows * a.wide;
    s.refs = s.lengths + a.rows;
    s.blocks = s.refs + a.pages;
    return s;
}

static PageScratch page_scratch(void* p, int64_t pages, int64_t rows, size_t* bytes)
{
    PageScratch w;
    w.list = (int32_t*)p;
    w.movers = w.list + pages;
    w.order = w.movers + pages;
    w.copies = (PageCopy*)(w.order + pages);
    w.count = (int32_t*)(w.copies + rows);
    if (bytes) *bytes = ((size_t)((uintptr_t)(w.count + 4) - (uintptr_t)p) + 15) & ~(size_t)15;
    return w;
}

static int64_t chunks_of(const fie_pages_args& a, const fie_cache_group& g)
{
    const int64_t bytes = (g.whole ? 1 : a.page) * g.token_bytes;
    // pieces that begin at 16-byte blocks need no chunk more than their bytes
    return (bytes + (g.shift ? 15 : 0) + kCopyChunk - 1) / kCopyChunk;
}

static int pages_check(const fie_pages_args* a, bool table)
{
    if (!a) return fail(FIE_E_ARG, "args is NULL");
    if (a->pages < 1 || a->pages > FIE_MAX_PAGES) return fail(FIE_E_ARG, "pages out of range [1, 2097152]");
    if (a->page < 1 || a->page > 65536) return fail(FIE_E_ARG, "page out of range [1, 65536]");
    if (a->group_count < 0 || a->group_count > FIE_MAX_CACHE_GROUPS) return fail(FIE_E_ARG, "group_count out of range [0, 8]");
    for (int i = 0; i < a->group_count; ++i) {
        const fie_cache_group& g = a->group[i];
        if (g.count < 0 || g.outer < 1 || g.token_bytes < 1 || g.token_bytes > 1 << 30 || (g.count && !g.base))
            return fail(FIE_E_ARG, "a cache group's layout is out of range");
        if ((int64_t)g.count * g.outer > kMostBlocks || chunks_of(*a, g) > kMostBlocks || (int64_t)g.count * g.outer * chunks_of(*a, g) > kMostBlocks)
            return fail(FIE_E_ARG, "a cache group's pages are too large");
    }
    if (!table) return FIE_OK;
    if (a->rows < 1 || a->rows > FIE_MAX_PAGE_ROWS) return fail(FIE_E_ARG, "rows out of range [1, 4096]");
    if (a->wide < 1 || a->wide > a->pages) return fail(FIE_E_ARG, "wide out of range [1, pages]");
    if (!a->state) return fail(FIE_E_ARG, "state is NULL");
    size_t need;
    page_scratch(nullptr, a->pages, a->rows, &need);
    if (!a->scratch || a->scratch_bytes < need) return fail(FIE_E_WORKSPACE, "scratch too small");
    if (((uintptr_t)a->scratch & 15) != 0) return fail(FIE_E_WORKSPACE, "scratch not 16-byte aligned");
    return FIE_OK;
}

// Copies of at most `most` pages, whose number may be known to the device alone.
static hipError_t copy_pages(const fie_pages_args& a, const PageList& l, int64_t most, hipStream_t st)
{
    for (int i = 0; i < a.group_count; ++i) {
        const fie_cache_group& g = a.group[i];
        if (!g.count || !most) continue;
        const int chunks = (int)chunks_of(a, g);
        const int64_t pieces = (int64_t)g.count * g.outer * chunks;
        // as many copies side by side as fill the CUs
        const int64_t side = std::min<int64_t>({most, 65535, std::max<int64_t>(1, (8 * std::max(cu_count(), 1) + pieces - 1) / pieces)});
        k_pages_copy<<<dim3((unsigned)pieces, (unsigned)side), kCopyThreads, 0, st>>>(l, g, a.page, chunks);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    return hipSuccess;
}

constexpr int kSmallTable = 8192;       // entries of a table that one workgroup forks

static hipError_t pages_step(const fie_pages_args& a, hipStream_t st)
{
    const PageState s = page_state(a);
    const PageScratch w = page_scratch(a.scratch, a.pages, a.rows, nullptr);
    const bool small = (int64_t)a.rows * a.wide <= kSmallTable;
    const bool moves = a.parents || a.lengths;          // whether any entry may change
    hipError_t e;
    if (!small && moves) {
        const int cols = a.rows <= 1024 ? 8 : 4;
        const size_t lds = (size_t)a.rows * (4 * cols + 4 + 2) + 4 * (size_t)s.nblocks;
        const unsigned grid = (unsigned)((a.wide + cols - 1) / cols);
        if (cols == 8) k_pages_fork<8><<<grid, kPageThreads, lds, st>>>(s, a.parents, a.lengths);
        else k_pages_fork<4><<<grid, kPageThreads, lds, st>>>(s, a.parents, a.lengths);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    const int bits = mark_bits(a.rows);
    const size_t area = std::max<size_t>(small ? (size_t)a.rows * a.wide : 0, (size_t)3 << bits);
    const size_t lds = ((size_t)3 * a.rows + s.nblocks + area) * 4;
    if (small && a.rows <= 64) k_pages_grow<true, 256><<<1, 256, lds, st>>>(s, w, a.parents, a.lengths, a.granted, bits, (int)area);
    else if (small) k_pages_grow<true, kPageThreads><<<1, kPageThreads, lds, st>>>(s, w, a.parents, a.lengths, a.granted, bits, (int)area);
    else k_pages_grow<false, kPageThreads><<<1, kPageThreads, lds, st>>>(s, w, a.parents, a.lengths, a.granted, bits, (int)area);
    e = hipGetLastError();
    if (e != hipSuccess || !a.lengths) return e;
    return copy_pages(a, PageList{w.copies, nullptr, nullptr, w.count, 0, a.pages}, a.rows, st);
}

static hipError_t pages_compact(const fie_pages_args& a, hipStream_t st)
{
    const PageState s = page_state(a);
    const PageScratch w = page_scratch(a.scratch, a.pages, a.rows, nullptr);
    hipError_t e;
    if (s.nblocks <= 2 && (int64_t)a.rows * a.wide <= kSmallTable) {
        k_pages_holes<true><<<1, kPageThreads, 0, st>>>(s, w, a.live);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    } else {
        k_pages_holes<false><<<(unsigned)s.nblocks, kPageThreads, 0, st>>>(s, w, a.live);
        if ((e = hipGetLastError()) != hipSuccess) return e;
        const int64_t entries = std::max((int64_t)a.rows * a.wide, (int64_t)a.pages / 2);
        k_pages_rename<<<(unsigned)std::min<int64_t>((entries + 255) / 256, 8 * std::max(cu_count(), 1)), 256, 0, st>>>(s, w);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    return copy_pages(a, PageList{nullptr, w.movers, w.list, w.count, 0, a.pages}, a.pages / 2, st);
}

}  // namespace fie

using namespace fie;

extern "C" size_t fie_pages_state_ints(int32_t pages, int32_t rows, int32_t wide)
{
    if (pages < 1 || pages > FIE_MAX_PAGES || rows < 1 || rows > FIE_MAX_PAGE_ROWS || wide < 1 || wide > pages) return 0;
    return (size_t)rows * wide + rows + pages + (pages + kPageBlock - 1) / kPageBlock;
}

extern "C" size_t fie_pages_scratch_bytes(int32_t pages, int32_t rows)
{
    if (pages < 1 || pages > FIE_MAX_PAGES || rows < 1 || rows > FIE_MAX_PAGE_ROWS) return 0;
    size_t bytes;
    page_scratch(nullptr, pages, rows, &bytes);
    return bytes;
}

extern "C" int fie_pages_step(const fie_pages_args* a, void* stream)
{
    if (const int rc = pages_check(a, true); rc != FIE_OK) return rc;
    if (!a->granted) return fail(FIE_E_ARG, "granted is NULL");
    return launch_status(pages_step(*a, (hipStream_t)stream), "k_pages_step");
}

extern "C" int fie_pages_compact(const fie_pages_args* a, void* stream)
{
    if (const int rc = pages_check(a, true); rc != FIE_OK) return rc;
    return launch_status(pages_compact(*a, (hipStream_t)stream), "k_pages_compact");
}

extern "C" int fie_pages_copy(const fie_pages_args* a, void* stream)
{
    if (const int rc = pages_check(a, false); rc != FIE_OK) return rc;
    if (a->copies < 0) return fail(FIE_E_ARG, "copies < 0");
    if (a->copies == 0) return FIE_OK;
    if (!a->src || !a->dst) return fail(FIE_E_ARG, "src or dst is NULL");
    return launch_status(copy_pages(*a, PageList{nullptr, a->src, a->dst, nullptr, a->copies, a->pages}, a->copies, (hipStream_t)stream),
                         "k_pages_copy");
}
