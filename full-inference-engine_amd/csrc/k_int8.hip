// The 8-bit integer product behind the C ABI of include/fie_ops.h: instantiations of int8.h's
// kernels and the choice among them.
#include <algorithm>

#include "int8.h"

namespace fie {

template <int DT, int MT, int NW, int S, int U>
static hipError_t rows_of(const fie_int8_args& a, int wide, hipStream_t st)
{
    k_int8_rows<DT, MT, NW, S, U><<<(a.n + 16 * NW - 1) / (16 * NW), 64 * S, 0, st>>>(a, wide);
    return hipGetLastError();
}

template <int DT, int BM, int BN, int WM, int WN, int NB, int KG, int OCC>
static hipError_t pipe_of(const fie_int8_args& a, int wide, hipStream_t st)
{
    const int64_t nrb = (a.m + BM - 1) / BM, ncb = (a.n + BN - 1) / BN;
    k_int8_pipe<DT, BM, BN, WM, WN, NB, KG, OCC><<<(unsigned)(8 * ((nrb * ncb + 7) / 8)), 64 * WM * WN * KG, 0, st>>>(a, (int)nrb, wide);
    return hipGetLastError();
}

// The pipe kernel's tiles, and what a CU takes for one of each, as measured at k 4096 (us, tiles as
// many as CUs, less the launch's own 3; then products on that tile, back to back with their launches,
// and in brackets the same on other tiles):
//   32 x 32, k in four groups    4.6   64 x 4096  7.4 (32 x 64 10.0, 64 x 64 12.6)
//   32 x 64                      6.5   16 x 151936  113 (64 x 64 124, 64 x 128 126)
//   64 x 64                     10.5   250 x 4096  13.1 (32 x 64 14.0, 64 x 128 17.3)
//   64 x 128                    17     128 x 16384  22.1 (64 x 64 26.2, 128 x 128 26.5)
//   128 x 128                   26     250 x 16384  29.0 (64 x 128 34.6, 256 x 128 38.5)
//   256 x 128                   40     256 x 151936  226 (256 x 256 254, 128 x 128 261)
//   256 x 256                   73     4096 x 4096 at k 16384  221 (256 x 128 261, 128 x 128 306)
// A product takes the tile with the least cost times rounds of the CUs; all of them go over k
// alike.
struct Tile { int bm, bn; float cost; };
constexpr Tile kTiles[] = {{32, 32, 4.6f}, {32, 64, 6.5f}, {64, 64, 10.5f}, {64, 128, 17.0f},
                           {128, 128, 26.0f}, {256, 128, 40.0f}, {256, 256, 73.0f}};

static int cus()
{
    const int n = cu_count();
    return n > 0 ? n : 256;
}

static int cheapest(int64_t m, int64_t n)
{
    const int64_t c = cus();
    int best = 0;
    float least = 0.0f;
    for (int i = 0; i < (int)(sizeof kTiles / sizeof kTiles[0]); ++i) {
        const Tile& t = kTiles[i];
        const int64_t tiles = ((m + t.bm - 1) / t.bm) * ((n + t.bn - 1) / t.bn);
        const float cost = t.cost * (float)((tiles + c - 1) / c);
        if (i == 0 || cost < least) { best = i; least = cost; }
    }
    return best;
}

// Rows that the pipe kernel's loads take: 16 bytes at aligned addresses, 32-bit offsets from a
// tile's first row.
static bool aligned_rows(const void* p, int64_t stride)
{
    return (((uintptr_t)p | (uint64_t)stride) & 15) == 0 && stride < (1 << 23);
}

// Tokens few enough to go with the weights at whatever address, straight to registers: us so and
// laid out first, 96 x 50001 at k 4097 159, 168; 128 x 5001 at k 1003 11.9, 16.0; but 128 x 20001 at
// k 4097 92, 75.
static bool by_rows(int64_t m, int n) { return m <= (n <= 2 * 16 * cus() ? 128 : 96); }

static int64_t pitch_of(int k) { return ((int64_t)k + kI8K - 1) / kI8K * kI8K; }

static size_t int8_workspace(const fie_int8_args& a)
{
    const bool ax = aligned_rows(a.x, a.x_stride), aw = aligned_rows(a.w, a.w_stride);
    if ((ax && aw) || by_rows(a.m, a.n)) return 0;
    return (size_t)((ax ? 0 : a.m) + (aw ? 0 : (int64_t)a.n)) * (size_t)pitch_of(a.k);
}

static hipError_t align_rows(const int8_t* src, int64_t stride, int64_t rows, int k, int8_t* dst, hipStream_t st)
{
    k_align_rows<<<(unsigned)((rows + 3) / 4), 256, 0, st>>>(src, stride, rows, k, dst, pitch_of(k));
    return hipGetLastError();
}

template <int DT>
static hipError_t int8_dt(fie_int8_args a, hipStream_t st)
{
    constexpr int SZ = DT == FIE_F32 ? 4 : 2;
    const int wide = ((uintptr_t)a.y % (4 * SZ)) == 0 && a.y_stride % 4 == 0;
    const bool ax = aligned_rows(a.x, a.x_stride), aw = aligned_rows(a.w, a.w_stride);
    if (!(ax && aw)) {
        if (by_rows(a.m, a.n)) {
            // 16 channels a workgroup up to one for each CU, where that is the shorter way; past it
            // 32, which save a round (and loads of the tokens), past two for each CU 64.  us, 16,
            // 32 and 64 channels:
            //    16 tokens   4096 at k 4097   7.8,  9.6         8190 at k 4097  13.8, 10.6
            //    32          4096 at k 4097  10.2, 12.6         9001 at k 4097  25.1, 23.7, 19.3
            //    64          4096 at k 1003   5.4,  6.4        20001 at k 4097  64.7, 52.3, 49.5
            //    77          4096 at k 1003   6.2,  7.5         5001 at k 4097  35.4, 21.7
            //   128          2000 at k 1003   7.5, 12.0         5001 at k 4097  47.6, 31.2
            const int per = (a.n - 1) / (16 * cus());
            if (a.m <= 16) return per ? rows_of<DT, 1, 2, 8, 1>(a, wide, st) : rows_of<DT, 1, 1, 8, 2>(a, wide, st);
            if (a.m <= 32)
                return per > 1 ? rows_of<DT, 2, 4, 8, 1>(a, wide, st)
                     : per     ? rows_of<DT, 2, 2, 8, 1>(a, wide, st)
                               : rows_of<DT, 2, 1, 8, 1>(a, wide, st);
            if (a.m <= 64)
                return per > 1 ? rows_of<DT, 4, 4, 8, 1>(a, wide, st)
                     : per     ? rows_of<DT, 4, 2, 8, 1>(a, wide, st)
                               : rows_of<DT, 4, 1, 8, 1>(a, wide, st);
            if (a.m <= 96) return per ? rows_of<DT, 6, 2, 8, 1>(a, wide, st) : rows_of<DT, 6, 1, 8, 1>(a, wide, st);
            return per ? rows_of<DT, 8, 2, 8, 1>(a, wide, st) : rows_of<DT, 8, 1, 8, 1>(a, wide, st);
        }
        int8_t* to = (int8_t*)a.workspace;
        hipError_t e = hipSuccess;
        if (!ax) {
            e = align_rows(a.x, a.x_stride, a.m, a.k, to, st);
            a.x = to;
            a.x_stride = pitch_of(a.k);
            to += a.m * a.x_stride;
        }
        if (e == hipSuccess && !aw) {
            e = align_rows(a.w, a.w_stride, a.n, a.k, to, st);
            a.w = to;
            a.w_stride = pitch_of(a.k);
        }
        if (e != hipSuccess) return e;
        if (!ax && !aw) a.k = (int)pitch_of(a.k);           // zeros on both sides: no last piece
    }
    switch (cheapest(a.m, a.n)) {
    case 0: return pipe_of<DT, 32, 32, 1, 2, 4, 4, 2>(a, wide, st);
    case 1: return pipe_of<DT, 32, 64, 1, 4, 4, 1, 3>(a, wide, st);
    case 2: return pipe_of<DT, 64, 64, 2, 2, 4, 1, 2>(a, wide, st);
    case 3: return pipe_of<DT, 64, 128, 2, 4, 3, 1, 4>(a, wide, st);
    case 4: return pipe_of<DT, 128, 128, 4, 4, 4, 1, 4>(a, wide, st);
    case 5: return pipe_of<DT, 256, 128, 4, 4, 3, 1, 4>(a, wide, st);
    default: return pipe_of<DT, 256, 256, 4, 4, 2, 1, 4>(a, wide, st);
    }
}

// A launch holds fewer than 2^32 threads (past that it leaves tiles out, without an error), so
// larger products go in pieces: channels and tokens whose layout (64 threads a row) and rows' kernel
// (32 a channel) fit, and tokens, whole tiles of any size, that leave 2^22 tiles of 32 x 32 (512
// threads each; larger tiles have at most twice the threads and half the tiles).
constexpr int64_t kMostChannels = 1 << 24, kMostTokens = 1 << 25, kMostTiles = 1 << 22;

static hipError_t int8_run(const fie_int8_args& a, hipStream_t st)
{
    const int64_t size = a.y_dtype == FIE_F32 ? 4 : 2;
    for (int64_t n0 = 0; n0 < a.n; n0 += kMostChannels) {
        fie_int8_args p = a;
        p.n = (int)std::min<int64_t>(a.n - n0, kMostChannels);
        p.w = a.w + n0 * a.w_stride;
        p.w_scale = a.w_scale + n0;
        p.bias = a.bias ? a.bias + n0 : nullptr;
        const int64_t most = std::min(kMostTokens, kMostTiles / ((p.n + 31) / 32) * 32 / 256 * 256);
        for (int64_t m0 = 0; m0 < a.m; m0 += most) {
            p.m = std::min(a.m - m0, most);
            p.x = a.x + m0 * a.x_stride;
            p.x_scale = a.x_scale + m0;
            p.y = (char*)a.y + (m0 * a.y_stride + n0) * size;
            hipError_t e;
            switch (a.y_dtype) {
            case FIE_F32: e = int8_dt<FIE_F32>(p, st); break;
            case FIE_F16: e = int8_dt<FIE_F16>(p, st); break;
            default: e = int8_dt<FIE_BF16>(p, st); break;
            }
            if (e != hipSuccess) return e;
        }
    }
    return hipSuccess;
}

static int int8_check(const fie_int8_args* a)
{
    if (!a) return fail(FIE_E_ARG, "args is NULL");
    if (a->m < 0 || a->m > 0x7FFFFF00 || a->n < 1 || a->n > 0x7FFFFF00) return fail(FIE_E_ARG, "sizes out of range");
    if (a->k < 1 || a->k > FIE_MAX_K) return fail(FIE_E_ARG, "k out of range [1, 131071]");
    if (a->y_dtype < FIE_F32 || a->y_dtype > FIE_BF16) return fail(FIE_E_ARG, "unknown dtype");
    if (a->x_stride < a->k || a->w_stride < a->k || a->y_stride < a->n) return fail(FIE_E_ARG, "a row stride is shorter than its row");
    if ((a->m + 31) / 32 * ((a->n + 31) / 32) > 0x0FFFFFFF) return fail(FIE_E_ARG, "m x n too large for one launch");
    if (a->m == 0) return FIE_OK;
    if (!a->x || !a->w || !a->x_scale || !a->w_scale || !a->y) return fail(FIE_E_ARG, "a required pointer is NULL");
    if (const size_t need = int8_workspace(*a)) {
        if (!a->workspace || a->workspace_bytes < need) return fail(FIE_E_WORKSPACE, "workspace too small for unaligned rows");
        if (((uintptr_t)a->workspace & 15) != 0) return fail(FIE_E_WORKSPACE, "workspace not 16-byte aligned");
    }
    return FIE_OK;
}

}  // namespace fie

using namespace fie;

extern "C" size_t fie_int8_workspace_size(const fie_int8_args* a)
{
    return a && a->m > 0 && a->n > 0 && a->k > 0 ? int8_workspace(*a) : 0;
}

extern "C" int fie_int8_linear(const fie_int8_args* a, void* stream)
{
    const int rc = int8_check(a);
    if (rc != FIE_OK || a->m == 0) return rc;
    return launch_status(int8_run(*a, (hipStream_t)stream), "k_int8");
}
