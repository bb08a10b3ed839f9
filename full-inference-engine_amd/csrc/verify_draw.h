// A row's draw in rank order (value descending, then index: the sampler's rule R4), its spans side
// by side, for rows without filters.  k_finish settles such a draw from its candidates, or takes
// the whole row through one workgroup where it lies deeper (a fifth of the draws at temperature 1
// on logits like a trained model's; about 90 us at vocab 151936 whatever else the step does).
//
// Three passes over the row, by radix on d = M - y: masses by bin of d, masses by part of the
// bin the draw lands in, then the tokens of that part.  Masses are the exact integers of rule R1
// (two limbs of 41 bits, added by atomics: no order).  After each pass the last workgroup to
// arrive looks for the draw.  What is left in the end is a short list, or one value that many
// tokens share (16-bit logits lie on a grid), whose tokens are then counted in index order; and
// for anything else a search over the keys by one workgroup.
//
// Three passes rather than one that keeps every token by bin: the row is 0.3 MB and stays in the
// caches, a list of its keys would be written and read at four times that.  The second and third
// read only tiles whose largest value reaches into the part.  Bound by latency and by the vector
// instructions of the masses (two 41-bit limbs a token): 123 draws of 151936 bf16 logits, the
// first pass within k_refused's 39 us, the second 11.6, the third 25.
#pragma once

namespace fie {

constexpr int kRankBins = 512;
constexpr int kRankList = kVerThreads;
constexpr int kRankTiles = 32;          // rows of fewer tiles have no room for the bins
constexpr uint64_t kLimb41 = (1ull << 41) - 1;

// In the last row's candidate slots: kRankTiles tiles hold 16 KiB.
struct RankState {
    uint64_t lo[kRankBins], hi[kRankBins];
    uint64_t list[kRankList];           // the last pass's tokens, (key, index) composites
    uint64_t goal[2];                   // what is left of the draw
    float M, f;                         // the row's maximum, bins a unit of d
    int32_t b1, b2;
    uint32_t n, kmin, kmax;             // tokens of the last pass, their keys
};
static_assert(sizeof(RankState) <= (size_t)kRankTiles * kCapW * 8, "the state fits its row's candidate slots");

FIE_DEV RankState* rank_state(const KParams& P, int row) { return (RankState*)(P.w.cand + (size_t)row * P.NT * kCapW); }

// The bin of a value and, within it, the part: both non-decreasing in d, ties in one.
FIE_DEV int rank_bin(float d, float f)
{
    const float q = d * f;
    return q < (float)(kRankBins - 1) ? (int)q : kRankBins - 1;
}
FIE_DEV int rank_part(float d, float f, int b)
{
    const float x = d * f - (float)b;                       // exact: f is a power of two
    const float q = b < kRankBins - 1 ? x * (float)kRankBins : x;      // the last bin has no end: whole bins
    return q < (float)(kRankBins - 1) ? (int)q : kRankBins - 1;
}

// The d of a bin, or of one of its parts: [lo, hi), exact ends.
struct RankRange { float lo, hi; };
FIE_DEV RankRange rank_range(int pass, float f, int b1, int b2)
{
    const bool end = b1 == kRankBins - 1;
    const float i = 1.0f / f;                               // a power of two
    if (pass == 1) return RankRange{-__builtin_inff(), __builtin_inff()};
    if (pass == 2) return RankRange{(float)b1 * i, end ? __builtin_inff() : (float)(b1 + 1) * i};
    const float lo = end ? (float)(b1 + b2) : (float)b1 + (float)b2 * (1.0f / kRankBins);
    const float hi = end ? (float)(b1 + b2 + 1) : (float)b1 + (float)(b2 + 1) * (1.0f / kRankBins);
    return RankRange{lo * i, end && b2 == kRankBins - 1 ? __builtin_inff() : hi * i};
}

// Clears a row's state, by one workgroup.  The bins span 8 times what the tiles' maxima do, 32 at
// most (below that lie weights of 2^-46 and less).
FIE_DEV void rank_begin(const KParams& P, int row, uint32_t* red)
{
    RankState& S = *rank_state(P, row);
    const int tid = threadIdx.x;
    const float* mt = P.w.mt + (size_t)row * (P.NT + 1);
    const float M = P.w.res[row].M;
    for (int i = tid; i < kRankBins; i += kVerThreads) { S.lo[i] = 0; S.hi[i] = 0; }
    const uint32_t k = tid < P.NT ? fkey(mt[1 + tid] + 0.0f) : 0xFFFFFFFFu;
    const float low = key_to_float(block_min_u32<kVerThreads>(k, red));
    if (tid == 0) {
        float span = 8.0f * (M - low);
        span = span > 0x1p-10f && span < 32.0f ? span : span < 32.0f && span > 0.0f ? 0x1p-10f : 32.0f;
        S.M = M;
        S.f = __uint_as_float(__float_as_uint((float)kRankBins / span) & 0x7F800000u);       // a power of two
        S.b1 = S.b2 = 0;
        S.n = 0;
        S.kmin = 0xFFFFFFFFu;
        S.kmax = 0;
        // the draw itself: floor(u T), exactly
        const RowRes& rr = P.w.res[row];
        S.goal[0] = rr.klo;
        S.goal[1] = rr.khi;
    }
}

FIE_DEV u128 rank_mass(float y, float m, uint64_t ct) { return mul64((uint64_t)__builtin_floorf(weight20(y - m) * 0x1p20f), ct); }

// Inclusive prefix sum of x in thread order, and the workgroup's total.
FIE_DEV u128 rank_scan(u128 x, u128* red, u128* total)
{
    u128 v = dwave_incl_scan_u128(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) red[threadIdx.x >> 6] = v;
    __syncthreads();
    u128 t = 0;
    for (int i = 0; i < kVerThreads / 64; ++i) {
        if (i < (int)(threadIdx.x >> 6)) v += red[i];
        t += red[i];
    }
    *total = t;
    return v;
}

// The bin in which `goal` lies, by the last workgroup; what is left goes to the state.
template <int PASS>
FIE_DEV void rank_find(RankState& S, u128 goal, u128* red)
{
    const int tid = threadIdx.x;
    static_assert(kRankBins == 2 * kVerThreads, "two bins a thread");
    u128 w[2], total;
#pragma unroll
    for (int i = 0; i < 2; ++i) w[i] = ((u128)from_all(&S.hi[2 * tid + i]) << 41) + from_all(&S.lo[2 * tid + i]);
    u128 before = rank_scan(w[0] + w[1], red, &total) - w[0] - w[1];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        S.lo[2 * tid + i] = 0;
        S.hi[2 * tid + i] = 0;
        if (before <= goal && goal < before + w[i]) {
            const u128 left = goal - before;
            S.goal[0] = (uint64_t)left;
            S.goal[1] = (uint64_t)(left >> 64);
            (PASS == 1 ? S.b1 : S.b2) = 2 * tid + i;
        }
        before += w[i];
    }
}

// One pass of one span; grid (spans, requests).
template <int DT, int PASS, int TPS>
FIE_DEV void rank_pass(const KParams& P, const VerWs& vw, int r, const VerJob& J, uint32_t* cnt)
{
    typedef SpanRow<DT, TPS> Row;
    constexpr int EPL = Row::EPL, WV = kVerThreads / 64, GPT = Row::GPT;
    __shared__ uint64_t blo[kRankBins], bhi[kRankBins];     // the last pass: the list, and its masses
    __shared__ u128 red[WV], left;
    __shared__ uint32_t flag, n, base, kmin, kmax, tiles[Row::TPS];
    const int tid = threadIdx.x, lane = tid & 63, V = P.a.vocab, spans = gridDim.x;
    const Row R(P, J.row, J.s, cnt);
    RankState& S = *rank_state(P, J.row);
    const float M = S.M, f = S.f;
    const int b1 = S.b1;
    const RankRange in = rank_range(PASS, f, b1, S.b2);
    const int lo = blockIdx.x * Row::kSpanV;
    if (PASS < 3)
        for (int i = tid; i < kRankBins; i += kVerThreads) { blo[i] = 0; bhi[i] = 0; }
    if (tid < Row::TPS) tiles[tid] = 0;
    if (tid == 0) { n = 0; kmin = 0xFFFFFFFFu; kmax = 0; }
    if (R.pen) R.count(lo);
    else __syncthreads();
    // a tile whose largest value is past the range has nothing in it (token 0's own tile aside)
    auto none = [&](int t0) { return t0 >= V || (t0 != 0 && M - R.mt[1 + t0 / kTile] >= in.hi); };
    auto inside = [&](float y, int idx) { const float d = M - y; return d >= in.lo && d < in.hi && idx < V; };
    auto mass = [&](float y, int idx, float m, uint64_t c) { return idx ? rank_mass(y, m, c) : mul64(1ull << 40, R.ct[0]); };
    float least = __builtin_inff(), most = -__builtin_inff();       // the last pass's values
    uint4 raw[Row::NL];
#pragma unroll
    for (int j = 0; j < Row::NL; ++j)
        if (!none(lo + j / GPT * kTile)) raw[j] = R.load(lo + (j * kVerThreads + tid) * EPL);
#pragma unroll
    for (int i = 0; i < Row::TPS; ++i) {
        const int t0 = lo + i * kTile;
        if (none(t0)) continue;
        const float m = R.mt[1 + t0 / kTile];
        const uint64_t c = R.ct[1 + t0 / kTile];
        uint32_t have = 0;                                  // of the wave's tokens
#pragma unroll
        for (int j = i * GPT; j < (i + 1) * GPT; ++j) {
            const int e0 = lo + (j * kVerThreads + tid) * EPL;
            float y[EPL];
            R.values(lo, e0, raw[j], y);
#pragma unroll
            for (int e = 0; e < EPL; ++e) {
                const bool is = inside(y[e], e0 + e);
                if (PASS < 3) {
                    if (!is) continue;
                    const u128 w = mass(y[e], e0 + e, m, c);
                    if (w == 0) continue;
                    const float d = M - y[e];
                    const int b = PASS == 1 ? rank_bin(d, f) : rank_part(d, f, b1);
                    atomicAdd((unsigned long long*)&blo[b], (unsigned long long)((uint64_t)w & kLimb41));
                    atomicAdd((unsigned long long*)&bhi[b], (unsigned long long)(uint64_t)(w >> 41));
                } else {
                    // a part's tokens only counted: masses are for the list and its ends (with
                    // them here, and an atomic a token, this pass took 44 us for 123 draws)
                    const uint64_t who = __ballot(is);
                    if (who == 0) continue;
                    have += popc64(who);
                    least = is ? __builtin_fminf(least, y[e]) : least;
                    most = is ? __builtin_fmaxf(most, y[e]) : most;
                    if (n < (uint32_t)kRankList) {          // still a list
                        uint32_t at = 0;
                        if (lane == (int)__builtin_ctzll(who)) at = atomicAdd(&n, popc64(who));
                        at = __shfl(at, (int)__builtin_ctzll(who), 64) + popc64(who & ((1ull << lane) - 1));
                        if (is && at < (uint32_t)kRankList) blo[at] = comp_key(fkey(y[e]), (uint32_t)(e0 + e));
                    }
                }
            }
        }
        if (PASS == 3 && lane == 0 && have) atomicAdd(&tiles[i], have);
    }
    if (PASS == 3) {
        const uint32_t a = dwave_min_u32(fkey(least)), b = dwave_max_u32(most > -__builtin_inff() ? fkey(most) : 0u);
        if (lane == 0 && b) {
            atomicMin(&kmin, a);
            atomicMax(&kmax, b);
        }
    }
    __syncthreads();
    uint64_t* const counts = vw.sum + (size_t)r * P.NT;     // the tiles' tokens in the part
    if (PASS < 3) {
        for (int i = tid; i < kRankBins; i += kVerThreads) {
            if (blo[i]) __hip_atomic_fetch_add(&S.lo[i], blo[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (bhi[i]) __hip_atomic_fetch_add(&S.hi[i], bhi[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    } else {
        uint32_t mine = 0;                                  // of the span
#pragma unroll
        for (int i = 0; i < Row::TPS; ++i) mine += tiles[i];
        if (tid == 0 && mine) {
            base = __hip_atomic_fetch_add(&S.n, mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_fetch_min(&S.kmin, kmin, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_fetch_max(&S.kmax, kmax, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        if (tid < Row::TPS && lo / kTile + tid < P.NT) to_all(&counts[lo / kTile + tid], (uint64_t)tiles[tid]);
        __syncthreads();
        if (mine <= (uint32_t)kRankList && (uint32_t)tid < mine && base + tid < (uint32_t)kRankList) to_all(&S.list[base + tid], blo[tid]);
    }
    if (!arrive_last(&vw.arrived[r], (uint32_t)spans, &flag)) return;

    if (tid == 0) vw.arrived[r] = 0;                        // for the next pass
    u128 goal = ((u128)S.goal[1] << 64) | S.goal[0];
    if (PASS < 3) {
        if (PASS == 1) goal = J.u < 1.0 ? floor_mul_f64(J.u, goal) : goal - 1;
        __syncthreads();
        rank_find<PASS>(S, goal, red);
        return;
    }
    // everything at once: the loads go past the caches
    const uint32_t total = from_all(&S.n), top = from_all(&S.kmax);
    uint32_t key = from_all(&S.kmin);
    const uint64_t entry = from_all(&S.list[tid]), count = from_all(&counts[min(tid, P.NT - 1)]);
    if (total <= (uint32_t)kRankList) {
        // a thread a token: the mass ranked before it
        const uint64_t c = (uint32_t)tid < total ? entry : 0ull;
        const uint32_t idx = comp_idx(c);
        u128 w = 0;
        if (c) w = mass(key_to_float(comp_k(c)), (int)idx, R.mt[1 + idx / kTile], R.ct[1 + idx / kTile]);
        u128* const ws = (u128*)bhi;
        static_assert(sizeof(bhi) >= kRankList * sizeof(u128), "the list's masses");
        blo[tid] = c;
        ws[tid] = w;
        __syncthreads();
        u128 before = 0;
        for (uint32_t i = 0; i < total; ++i)
            if (blo[i] > c) before += ws[i];
        if (c && before <= goal && goal < before + w) *J.out = (int64_t)idx;
        return;
    }
    int first = 0;                                          // tokens before it are ruled out
    if (key == top) {
        // one value: its mass in a tile, times the tile's tokens (token 0 is not among the
        // first tile's: it goes by its own scale)
        const float y = key_to_float(key);
        u128 x = 0, all;
        if (tid < P.NT) {
            uint64_t k = count;
            if (tid == 0 && inside(R.m0, 0)) { --k; x = mul64(1ull << 40, R.ct[0]); }
            if (k) x += rank_mass(y, R.mt[1 + tid], R.ct[1 + tid]) * k;
        }
        const u128 incl = rank_scan(x, red, &all);
        if (incl - x <= goal && goal < incl) {
            base = (uint32_t)tid;
            left = goal - (incl - x);
        }
        __syncthreads();
        first = (int)base * kTile;
        goal = left;
    } else {
        // many tokens of several values: the value by a search over the keys
        auto at_least = [&](uint32_t k) {
            u128 sum = 0, all;
            for (int t0 = 0; t0 < V; t0 += kTile) {
                if (none(t0)) continue;
                if (R.pen) R.count(t0);
                for (int j = 0; j < GPT; ++j) {
                    const int e0 = t0 + (j * kVerThreads + tid) * EPL;
                    float y[EPL];
                    R.values(t0, e0, R.load(e0), y);
                    for (int e = 0; e < EPL; ++e)
                        if (inside(y[e], e0 + e) && fkey(y[e]) >= k) sum += mass(y[e], e0 + e, R.mt[1 + t0 / kTile], R.ct[1 + t0 / kTile]);
                }
            }
            rank_scan(sum, red, &all);
            return all;
        };
        uint32_t hi = top + 1;                              // at_least(key) > goal >= at_least(hi)
        while (hi - key > 1) {
            const uint32_t mid = key + (hi - key) / 2;
            if (at_least(mid) > goal) key = mid;
            else hi = mid;
        }
        goal -= at_least(key + 1);
    }
    for (int t0 = first; t0 < V; t0 += kTile) {
        if (none(t0)) continue;
        if (R.pen) R.count(t0);
        for (int j = 0; j < GPT; ++j) {
            const int e0 = t0 + (j * kVerThreads + tid) * EPL;
            float y[EPL];
            u128 w[EPL], mine = 0, sum;
            R.values(t0, e0, R.load(e0), y);
#pragma unroll
            for (int e = 0; e < EPL; ++e) {
                w[e] = e0 + e < V && fkey(y[e]) == key ? mass(y[e], e0 + e, R.mt[1 + t0 / kTile], R.ct[1 + t0 / kTile]) : 0;
                mine += w[e];
            }
            u128 b = rank_scan(mine, red, &sum) - mine;
            if (b <= goal && goal < b + mine) {             // one thread
#pragma unroll
                for (int e = 0; e < EPL; ++e) {
                    if (b <= goal && goal < b + w[e]) *J.out = e0 + e;
                    b += w[e];
                }
            }
            if (goal < sum) return;                         // the same in every thread
            goal -= sum;
        }
    }
}

template <int DT, int PASS, int TPS>
__global__ __launch_bounds__(kVerThreads) void k_rank(const KParams P, const VerWs vw)
{
    extern __shared__ uint32_t cnt[];       // a span's, with penalties
    const VerJob J = vw.job[blockIdx.y];
    if (J.row < 0 || J.lim != kRankDraw) return;
    rank_pass<DT, PASS, TPS>(P, vw, blockIdx.y, J, cnt);
}

}  // namespace fie
