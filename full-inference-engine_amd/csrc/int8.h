// The matrix product in 8-bit integers with scales for each token and channel
// (fie_int8_linear): y = x_scale w_scale sum_k x w + bias.
#pragma once

#include <type_traits>

#include "launchers.h"
#include "fie_ops.h"

namespace fie {

typedef int32_t i32x4_t __attribute__((ext_vector_type(4)));

// D += A (16 x 64) B (64 x 16) in int32.  Lane l supplies 16 consecutive k of A's row l % 16
// and of B's column l % 16, k-group l / 16, and receives D rows 4 (l / 16) .. +3 of column
// l % 16.  Whatever order the instruction pairs k in, A and B take it alike.
FIE_DEV i32x4_t mfma_i8(i32x4_t a, i32x4_t b, i32x4_t c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }

template <int DT>
FIE_DEV uint16_t round16(float v)
{
    if constexpr (DT == FIE_BF16) return __builtin_bit_cast(uint16_t, (__bf16)v);
    else return __builtin_bit_cast(uint16_t, (_Float16)v);
}

// Four neighbouring channels of one token, scaled, from n on: one store where `wide` (rows of
// y aligned to four elements) and all four are inside.
template <int DT>
FIE_DEV void store_scaled(const fie_int8_args& a, int64_t m, int n, i32x4_t acc, float xs, bool wide)
{
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = min(n + i, a.n - 1);
        v[i] = (float)acc[i] * xs * a.w_scale[c];
        if (a.bias) v[i] += a.bias[c];
    }
    if constexpr (DT == FIE_F32) {
        float* p = (float*)a.y + m * a.y_stride + n;
        if (wide && n + 4 <= a.n) *(float4*)p = make_float4(v[0], v[1], v[2], v[3]);
        else
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < a.n) p[i] = v[i];
    } else {
        uint16_t* p = (uint16_t*)a.y + m * a.y_stride + n;
        uint32_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = round16<DT>(v[i]);
        if (wide && n + 4 <= a.n) *(uint2*)p = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
        else
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < a.n) p[i] = (uint16_t)h[i];
    }
}

constexpr int kI8K = 128;               // bytes of k a stage

// Chunk c (of 8) of operand row n sits at slot n * 8 + (c ^ (n & 7)): the eight lanes one LDS
// cycle serves read eight rows' chunk c from eight distinct bank groups.
FIE_DEV int i8_slot(int n, int c) { return n * 8 + (c ^ (n & 7)); }

// 16 bytes at any address: the 16 from the word that holds the first, the word after them, and a
// shift.  (One load at the byte's own address takes 3 times as long: 16 x 50001 at k 4097 151 us.)
// Only words that hold some of the 16 bytes are touched.
struct Any16 {
    typedef uint32_t raw __attribute__((ext_vector_type(4), aligned(4)));
    raw r;
    uint32_t e;
    FIE_DEV void load(const int8_t* p, uint32_t sh)         // sh: the low two bits of p
    {
        const int8_t* b = p - sh;
        r = *(const raw*)b;
        e = *(const uint32_t*)(b + (sh ? 16 : 12));
    }
    FIE_DEV i32x4_t get(uint32_t sh) const
    {
        return i32x4_t{(int32_t)__builtin_amdgcn_alignbyte(r.y, r.x, sh), (int32_t)__builtin_amdgcn_alignbyte(r.z, r.y, sh),
                       (int32_t)__builtin_amdgcn_alignbyte(r.w, r.z, sh), (int32_t)__builtin_amdgcn_alignbyte(e, r.w, sh)};
    }
};
FIE_DEV uint32_t low2(const int8_t* p) { return (uint32_t)(uintptr_t)p & 3u; }

// 16 bytes of a row of at least 16 from k0 on; those at or past K are 0.  Where the row ends inside
// them, its last 16 bytes are loaded and shifted down, on no branch.
struct Last16 {
    Any16 v;
    uint32_t sh;
    int past;
    FIE_DEV void load(const int8_t* rowp, int k0, int K)
    {
        const int8_t* p = rowp + min(k0, K - 16);
        past = min(max(k0 + 16 - K, 0), 16);
        sh = low2(p);
        v.load(p, sh);
    }
    FIE_DEV i32x4_t get() const
    {
        const i32x4_t r = v.get(sh);
        const u128 x = ((u128)(uint32_t)r.w << 96) | ((u128)(uint32_t)r.z << 64) | ((u128)(uint32_t)r.y << 32) | (uint32_t)r.x;
        const u128 t = past < 16 ? x >> (8 * past) : 0;
        return i32x4_t{(int32_t)(uint32_t)t, (int32_t)(uint32_t)(t >> 32), (int32_t)(uint32_t)(t >> 64), (int32_t)(uint32_t)(t >> 96)};
    }
};

// The same of a row shorter than 16.
FIE_DEV i32x4_t load_short(const int8_t* rowp, int k0, int K)
{
    i32x4_t r{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const uint32_t b = (uint8_t)rowp[min(k0 + i, K - 1)];
        r[i / 4] |= (int32_t)((k0 + i < K ? b : 0u) << (8 * (i % 4)));
    }
    return r;
}

// A wave's 128 bytes of 16 rows at any address: lane l holds bytes 64 h + 16 (l / 16) .. +15 of
// row l % 16.  Each lane loads the 16 from the word that holds its first; the word after them is
// the first of the lane 16 further on (or of the other half, or one more load), so that no byte is
// loaded twice: with a load of its own for each such word the lines were out of the L1 again
// before it came (16 x 50001 at k 4097 73 us against 60).
struct Chunk {
    Any16::raw r[2];
    uint32_t e;
    FIE_DEV void load(const int8_t* p, const int8_t* past)      // p: a multiple of 4
    {
        r[0] = *(const Any16::raw*)p;
        r[1] = *(const Any16::raw*)(p + 64);
        e = *(const uint32_t*)past;
    }
    template <int H> FIE_DEV i32x4_t get(uint32_t sh, int lane) const
    {
        const uint32_t x = lane < 16 ? (H == 0 ? r[1].x : e) : r[H].x;
        const uint32_t n = (uint32_t)__builtin_amdgcn_ds_bpermute(((lane + 16) & 63) * 4, (int)x);
        const Any16 v{r[H], n};
        return v.get(sh);
    }
};

// Rows at any address into rows of whole stages at aligned ones, 0 past k: what the pipe kernel
// needs.  A wave a row; a lane makes a word from the two that hold its bytes, so that every
// load and store of a wave is one piece of 256 bytes (16 bytes a lane at odd addresses take
// four times as long).  250 x 16384 at k 4097 52 us with this, the product alone 29.  Bound by HBM: the matrix
// read and written once, on top of what the product reads.
__global__ __launch_bounds__(256) void k_align_rows(const int8_t* src, int64_t stride, int64_t rows, int K, int8_t* dst, int64_t pitch)
{
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    const int8_t* p = src + row * stride;
    const uint32_t sh = (uint32_t)(uintptr_t)p & 3u;
    const uint32_t* b = (const uint32_t*)(p - sh);
    const int words = (int)((sh + K + 3) / 4);          // that hold some of the row
    uint32_t* out = (uint32_t*)(dst + row * pitch);
    constexpr int U = 4;                                // words of a lane on their way together
    for (int j0 = lane; j0 < (int)(pitch / 4); j0 += 64 * U) {
        uint32_t lo[U], hi[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            lo[u] = b[min(j0 + 64 * u, words - 1)];
            hi[u] = b[min(j0 + 64 * u + 1, words - 1)];
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + 64 * u;
            uint32_t v = __builtin_amdgcn_alignbyte(hi[u], lo[u], sh);
            const int left = K - 4 * j;                 // bytes of the row from this word on
            if (left < 4) v = left > 0 ? v & ((1u << (8 * left)) - 1u) : 0u;
            if (j < (int)(pitch / 4)) out[j] = v;
        }
    }
}

// Few tokens: bound by the weights' way from memory.  A workgroup takes 16 NW channels and all
// tokens, 16 MT at most; its S waves take k in turn, 128 bytes each (whole lines of 16 NW rows),
// U of them loaded at once straight into the matrix instructions' operands, with no LDS and no
// barrier before the waves' sums meet.  For rows that the pipe kernel's loads do not take: 16
// bytes at any address take shifts and a word of a neighbour's, and rows straddle lines, so it stays below
// the memory's rate (16 x 50001 at k 4097 50 us, 4.1 TB/s; with the weights' rows padded to 16 bytes
// 43, and 38 by the pipe kernel with the tokens' as well).
template <int DT, int MT, int NW, int S, int U>
__global__ __launch_bounds__(64 * S) void k_int8_rows(const fie_int8_args a, int wide)
{
    __shared__ i32x4_t red[S][MT * NW][64];
    const int lane = threadIdx.x & 63, K = a.k;
    const int s = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * (16 * NW);
    const int8_t* wp[NW];
    const int8_t* xp[MT];
#pragma unroll
    for (int q = 0; q < NW; ++q) wp[q] = a.w + (int64_t)min(n0 + 16 * q + (lane & 15), a.n - 1) * a.w_stride + 16 * (lane >> 4);
#pragma unroll
    for (int m = 0; m < MT; ++m) xp[m] = a.x + min((int64_t)(16 * m + (lane & 15)), a.m - 1) * a.x_stride + 16 * (lane >> 4);
    i32x4_t acc[MT][NW];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int q = 0; q < NW; ++q) acc[m][q] = i32x4_t{0, 0, 0, 0};
    const int at = 16 * (lane >> 4);
    uint32_t ws[NW], xs[MT];
    const int8_t *we[NW], *xe[MT];                  // the word past the row's 128 bytes that holds some of them, or the last
    auto past = [&](const int8_t* p, uint32_t sh) { return p - at - sh + (sh ? 128 : 124); };
#pragma unroll
    for (int q = 0; q < NW; ++q) { ws[q] = low2(wp[q]); we[q] = past(wp[q], ws[q]); }
#pragma unroll
    for (int m = 0; m < MT; ++m) { xs[m] = low2(xp[m]); xe[m] = past(xp[m], xs[m]); }
    // Loads first, then what uses them: left to itself the compiler waits for each before the next.
    auto steps = [&](int k0, auto count) {          // chunks k0, k0 + 128 S, ..
        constexpr int N = decltype(count)::value;
        Chunk fw[N][NW], fx[N][MT];
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int k = k0 + u * (128 * S);
#pragma unroll
            for (int q = 0; q < NW; ++q) fw[u][q].load(wp[q] - ws[q] + k, we[q] + k);
#pragma unroll
            for (int m = 0; m < MT; ++m) fx[u][m].load(xp[m] - xs[m] + k, xe[m] + k);
        }
        __builtin_amdgcn_sched_barrier(0);
        auto half = [&](auto which, int u) {
            constexpr int H = decltype(which)::value;
            i32x4_t w[NW];
#pragma unroll
            for (int q = 0; q < NW; ++q) w[q] = fw[u][q].template get<H>(ws[q], lane);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const i32x4_t x = fx[u][m].template get<H>(xs[m], lane);
#pragma unroll
                for (int q = 0; q < NW; ++q) acc[m][q] = mfma_i8(w[q], x, acc[m][q]);
            }
        };
#pragma unroll
        for (int u = 0; u < N; ++u) {
            half(std::integral_constant<int, 0>{}, u);
            half(std::integral_constant<int, 1>{}, u);
        }
    };
    const int full = K / 128;                       // whole chunks
    int c = s;
    for (; c + (U - 1) * S < full; c += U * S) steps(c * 128, std::integral_constant<int, U>{});
    for (; c < full; c += S) steps(c * 128, std::integral_constant<int, 1>{});
    if (c == full && K < 16) {                      // the rest, by the wave whose turn it is
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int q = 0; q < NW; ++q) acc[m][q] = mfma_i8(load_short(wp[q] - at, at, K), load_short(xp[m] - at, at, K), acc[m][q]);
    } else if (c == full) {
#pragma unroll 1
        for (int k0 = full * 128; k0 < K; k0 += 64) {
            Last16 fw[NW], fx[MT];
#pragma unroll
            for (int q = 0; q < NW; ++q) fw[q].load(wp[q] - at, k0 + at, K);
#pragma unroll
            for (int m = 0; m < MT; ++m) fx[m].load(xp[m] - at, k0 + at, K);
            __builtin_amdgcn_sched_barrier(0);
            i32x4_t w[NW];
#pragma unroll
            for (int q = 0; q < NW; ++q) w[q] = fw[q].get();
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const i32x4_t x = fx[m].get();
#pragma unroll
                for (int q = 0; q < NW; ++q) acc[m][q] = mfma_i8(w[q], x, acc[m][q]);
            }
        }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int q = 0; q < NW; ++q) red[s][m * NW + q][lane] = acc[m][q];
    __syncthreads();
    for (int f = s; f < MT * NW; f += S) {
        i32x4_t t = red[0][f][lane];
#pragma unroll
        for (int i = 1; i < S; ++i) t += red[i][f][lane];
        const int64_t row = 16 * (f / NW) + (lane & 15);
        const int n = n0 + 16 * (f % NW) + 4 * (lane >> 4);
        if (row < a.m && n < a.n) store_scaled<DT>(a, row, n, t, a.x_scale[row], wide);
    }
}

// Many tokens: BM tokens by BN channels a workgroup of WM x WN waves.  k goes in stages of 128
// bytes through NB LDS buffers that the loads fill by themselves (16 bytes a lane, no registers
// between), NB - 1 stages ahead; a stage costs one barrier.  A wave's instruction fills eight
// rows of 128 bytes in lane order, so the swizzle of i8_slot is in the addresses it loads from.
// Large products are bound by the matrix cores and the LDS that feeds them (4096 x 4096 at k 16384
// 216-226 us, 2.4-2.5 Pop/s, 16 waves of 64 x 64: 8 waves 242, 128 x 128 306), few tokens by the
// weights' way from memory (16 x 151936 at k 4096 111-114 us, 5.5 TB/s), and what lies between by
// the loads into LDS, 55-60 GB/s a CU (250 x 16384 at k 4096 25-26 us a dispatch, 28.6 with the
// launch, where operations and bytes alone take 14; more buffers, fewer waves, two stages a barrier took as long or longer).
typedef __attribute__((address_space(3))) void* lds_ptr;

// Workgroup b's tile of nrb x ncb.  Workgroups are dealt to the eight XCDs round robin: each
// XCD takes an eighth of the tiles, in bands of kBand token blocks down and then across, so
// that the tiles it works on at a time share their rows in its L2.  Grid: tile_grid().
constexpr int kBand = 4;
FIE_DEV bool tile_at(int b, int nrb, int ncb, int* rb, int* cb)
{
    const int total = nrb * ncb, share = (total + 7) / 8;
    const int j = b >> 3, id = (b & 7) * share + j;
    if (j >= share || id >= total) return false;
    const int band = id / (kBand * ncb), in = id - band * (kBand * ncb);
    const int h = min(kBand, nrb - band * kBand);
    *rb = band * kBand + in % h;
    *cb = in / h;
    return true;
}

// All but the wave's last N loads into LDS are done, and all that it reads from there.
template <int N> FIE_DEV void wait_loads() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory"); }

FIE_DEV void meet()             // a barrier that waits for no load
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// KG groups of WM x WN waves take the stages in turn, each in buffers of its own, and their sums
// meet at the end: more of them in flight where there are few tiles.
template <int DT, int BM, int BN, int WM, int WN, int NB, int KG, int OCC>
__global__ __launch_bounds__(64 * WM * WN * KG, OCC) void k_int8_pipe(const fie_int8_args a, int nrb, int wide)
{
    constexpr int NWV = WM * WN;                                // waves of a group
    constexpr int FM = BM / WM / 16, FN = BN / WN / 16;         // 16 x 16 results of a wave
    constexpr int ROWS = BM + BN, NI = ROWS / 8 / NWV;          // loads of a wave a stage
    static_assert(ROWS % (8 * NWV) == 0 && BM % 8 == 0, "whole loads");
    static_assert(NB * ROWS * kI8K >= BM * BN * 4 || KG == 1, "a group's sums fit its buffers");
    __shared__ __attribute__((aligned(1024))) int8_t L[KG][NB][ROWS * kI8K];
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), grp = wv / NWV, wave = wv % NWV;
    int rb, cb;
    if (!tile_at(blockIdx.x, nrb, (a.n + BN - 1) / BN, &rb, &cb)) return;
    const int t0 = cb * BN;
    const int64_t r0 = (int64_t)rb * BM;
    // load i of this wave: rows 8 (wave + NWV i) .. +7 of the stage (tokens, then channels)
    uint32_t off[NI];
    const int8_t* const xb = a.x + r0 * a.x_stride;
    const int8_t* const wb = a.w + (int64_t)t0 * a.w_stride;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int r = 8 * (wave + NWV * i) + (lane >> 3), c = (lane & 7) ^ (r & 7);
        const int rm = (int)min((int64_t)r, a.m - 1 - r0), rn = min(r - BM, a.n - 1 - t0);
        off[i] = (r < BM ? (uint32_t)rm * (uint32_t)a.x_stride : (uint32_t)rn * (uint32_t)a.w_stride) + 16u * c;
    }
    auto issue = [&](int s) {                                   // the group's s-th stage
        int8_t* to = L[grp][s % NB];
        const int64_t k0 = (int64_t)(s * KG + grp) * kI8K;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int at = wave + NWV * i;
            const int8_t* b = (8 * at < BM ? xb : wb) + k0;
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(b + off[i]), (lds_ptr)(to + at * 1024), 16, 0, 0);
        }
    };
    const int wr = wave % WM, wn = wave / WM;
    i32x4_t acc[FM][FN];
#pragma unroll
    for (int m = 0; m < FM; ++m)
#pragma unroll
        for (int q = 0; q < FN; ++q) acc[m][q] = i32x4_t{0, 0, 0, 0};
    auto mul = [&](const int8_t* b) {
        const i32x4_t* l = (const i32x4_t*)b;
#pragma unroll
        for (int kk = 0; kk < kI8K / 64; ++kk) {
            const int c = kk * 4 + (lane >> 4);
            i32x4_t fx[FM], fw[FN];
#pragma unroll
            for (int m = 0; m < FM; ++m) fx[m] = l[i8_slot((BM / WM) * wr + 16 * m + (lane & 15), c)];
#pragma unroll
            for (int q = 0; q < FN; ++q) fw[q] = l[i8_slot(BM + (BN / WN) * wn + 16 * q + (lane & 15), c)];
#pragma unroll
            for (int m = 0; m < FM; ++m)
#pragma unroll
                for (int q = 0; q < FN; ++q) acc[m][q] = mfma_i8(fw[q], fx[m], acc[m][q]);
        }
    };
    const int full = a.k / kI8K;                                // whole stages
    const int ns = (full - grp + KG - 1) / KG;                  // this group's
    const int most = (full + KG - 1) / KG;                      // the first group's: no group has more
#pragma unroll
    for (int s = 0; s < NB - 1; ++s)
        if (s < ns) issue(s);
    for (int s = 0; s < most; ++s) {
        // this stage's loads of every wave are done, and every wave is past the stage before
        if (s + NB - 1 <= ns) wait_loads<(NB - 2) * NI>();
        else wait_loads<0>();
        meet();
        if (s + NB - 1 < ns) issue(s + NB - 1);
        if (KG == 1 || s < ns) mul(L[grp][s % NB]);
    }
    if (a.k % kI8K) {                                           // the rest of k, 0 past its end
        __syncthreads();
        if (grp == 0) {
            const int8_t* row[NI];
            int k0[NI];
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int r = 8 * (wave + NWV * i) + (lane >> 3), c = (lane & 7) ^ (r & 7);
                row[i] = (8 * (wave + NWV * i) < BM ? xb : wb) + (off[i] - 16u * c);
                k0[i] = full * kI8K + 16 * c;
            }
            auto put = [&](int i, i32x4_t v) { *(i32x4_t*)(L[0][0] + (wave + NWV * i) * 1024 + lane * 16) = v; };
            if (a.k < 16) {
#pragma unroll
                for (int i = 0; i < NI; ++i) put(i, load_short(row[i], k0[i], a.k));
            } else {                                            // the loads together
                Last16 v[NI];
#pragma unroll
                for (int i = 0; i < NI; ++i) v[i].load(row[i], k0[i], a.k);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < NI; ++i) put(i, v[i].get());
            }
        }
        __syncthreads();
        if (grp == 0) mul(L[0][0]);
    }
    if constexpr (KG > 1) {                                     // the groups' sums
        __syncthreads();
        i32x4_t* mine = (i32x4_t*)L[grp][0];
        if (grp)
#pragma unroll
            for (int m = 0; m < FM; ++m)
#pragma unroll
                for (int q = 0; q < FN; ++q) mine[((wave * FM + m) * FN + q) * 64 + lane] = acc[m][q];
        __syncthreads();
        if (grp) return;
#pragma unroll
        for (int g = 1; g < KG; ++g) {
            const i32x4_t* other = (const i32x4_t*)L[g][0];
#pragma unroll
            for (int m = 0; m < FM; ++m)
#pragma unroll
                for (int q = 0; q < FN; ++q) acc[m][q] += other[((wave * FM + m) * FN + q) * 64 + lane];
        }
    }
#pragma unroll
    for (int m = 0; m < FM; ++m) {
        const int64_t row = r0 + (BM / WM) * wr + 16 * m + (lane & 15);
        if (row >= a.m) continue;
        const float xs = a.x_scale[row];
#pragma unroll
        for (int q = 0; q < FN; ++q) {
            const int n = t0 + (BN / WN) * wn + 16 * q + 4 * (lane >> 4);
            if (n < a.n) store_scaled<DT>(a, row, n, acc[m][q], xs, wide);
        }
    }
}

}  // namespace fie
