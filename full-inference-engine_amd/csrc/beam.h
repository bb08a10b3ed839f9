// Beam search's selection (fie_beam_step): the best continuations of a request's beams.
#pragma once

#include "copy.h"
#include "launchers.h"
#include "fie_decode.h"

namespace fie {

constexpr int kBeamThreads = 256, kBeamWaves = kBeamThreads / 64;
constexpr int kBeamEach = 32;                           // logits of a thread a tile
constexpr int kBeamTile = kBeamThreads * kBeamEach;
constexpr int kBeamList = 1024;                         // candidates a workgroup holds,
constexpr int kBeamShare = kBeamList / kBeamWaves;      // and a wave
constexpr int kBeamSpans = 32;                          // most spans of a row
constexpr float kLog2e = 1.44269502f;
constexpr float kLargest = 3.40282347e38f;

// A span's results: the largest logit, the sum of exp(x - it), how many candidates.
struct BeamSpan {
    double sum;
    float top;
    int32_t count;
};

// The workspace: spans' results, then their candidates, best first.
struct BeamWork {
    BeamSpan* span;             // [rows][spans]
    uint64_t* cand;             // [rows][spans][most]
    int spans, tiles, most;     // of a row; tiles of a span; candidates of a span
};

FIE_DEV float beam_clean(float x) { return x != x ? -__builtin_inff() : __builtin_fminf(x, kLargest); }

template <int DT> struct BeamVec {                      // 16 bytes of logits
    static constexpr int N = DT == FIE_F32 ? 4 : 8;
    static FIE_DEV void open(const vec4_t& r, float* x)
    {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == FIE_F32) x[i] = __uint_as_float(w[i]);
            else if constexpr (DT == FIE_BF16) {
                x[2 * i] = __uint_as_float(w[i] << 16);
                x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
            } else {
                x[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)w[i]);
                x[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i] >> 16));
            }
        }
    }
};

// The largest key T, low LOW bits 0, that at least `rank` lanes of the wave reach.  (A logit's upper
// half has 7 bits behind the point's; a total's upper word needs its lower bits: by 16 of them the
// bound was 2 below totals about -40, and ten times the candidates were ranked.)
template <int LOW> FIE_DEV uint32_t beam_reach(uint32_t key, int rank)
{
    uint32_t t = 0;
#pragma unroll
    for (int bit = 31; bit >= LOW; --bit) {
        const uint32_t up = t | (1u << bit);
        if (__popcll(__ballot(key >= up)) >= rank) t = up;
    }
    return t;
}

FIE_DEV bool beam_dead(const fie_beam_args& a, int row)
{
    return a.done[row / a.beams] || !(a.scores[row] > -__builtin_inff());
}

// A row's logits in vectors at aligned addresses; those of the first and the last vector that
// are outside the row count as -inf (no vector without some of the row is touched).
template <int DT> struct BeamRow {
    static constexpr int N = BeamVec<DT>::N, LOADS = kBeamEach / N;
    const vec4_t* base;
    int shift, vocab, vecs;
    FIE_DEV BeamRow(const fie_beam_args& a, int row)
    {
        constexpr int SZ = 16 / N;
        const uintptr_t p = (uintptr_t)a.logits + (uintptr_t)((int64_t)row * a.row_stride * SZ);
        base = (const vec4_t*)(p & ~(uintptr_t)15);
        shift = (int)(p & 15) / SZ;
        vocab = a.vocab;
        vecs = (shift + vocab + N - 1) / N;
    }
    FIE_DEV void load(int tile, vec4_t (&r)[LOADS]) const
    {
#pragma unroll
        for (int j = 0; j < LOADS; ++j) r[j] = global_get<vec4_t>(base + min((tile * LOADS + j) * kBeamThreads + (int)threadIdx.x, vecs - 1));
    }
    FIE_DEV int index(int tile, int e) const            // of the thread's e-th logit of a tile
    {
        return ((tile * LOADS + e / N) * kBeamThreads + (int)threadIdx.x) * N + e % N - shift;
    }
    FIE_DEV void open(int tile, const vec4_t (&r)[LOADS], float (&x)[kBeamEach]) const
    {
#pragma unroll
        for (int j = 0; j < LOADS; ++j) BeamVec<DT>::open(r[j], x + j * N);
        if (tile == 0 || (tile + 1) * LOADS * kBeamThreads >= vecs)
#pragma unroll
            for (int e = 0; e < kBeamEach; ++e) {
                const int i = index(tile, e);
                if (i < 0 || i >= vocab) x[e] = -__builtin_inff();
            }
    }
};

// Workgroups of a CU at a time.
template <int DT> constexpr int kBeamHold = DT == FIE_BF16 ? 5 : 4;

struct BeamShared {
    union {
        uint64_t list[kBeamList];
        uint32_t hist[2048];        // of radix passes, before the list is made
    };
    uint32_t wave[kBeamWaves];
    double sum[kBeamWaves];
    float top[kBeamWaves];
    int32_t count, held[kBeamWaves];
    uint32_t above, bin;
};

// The `need`-th best candidate of a span, exactly: radix passes over (key, index) that read the
// span again, and at the end the `need` best into the list.  For spans whose candidates do not
// fit the list: equal logits, logits in rising order, and spans whose first tile leaves a wave without
// logits, so that nothing bounds them.  With few rows a span is a tile, and a row's last tile of fewer
// than 193 vectors is such a one: 4 rows of 50257 in bf16 19 us, of 57344 (7 whole tiles) 7.  (In line: a call takes stack in memory,
// and with it 20 us between launches.)
template <int DT>
FIE_DEV int beam_deep(const BeamRow<DT>& row, int first, int last, int most, BeamShared& S)
{
    const int tid = threadIdx.x;
    auto each = [&](auto&& f) {
        constexpr int N = BeamRow<DT>::N, LOADS = BeamRow<DT>::LOADS;
#pragma unroll 1
        for (int j = first * LOADS; j < min(last * LOADS, (row.vecs + kBeamThreads - 1) / kBeamThreads); ++j) {
            const int v = j * kBeamThreads + tid;
            float x[N];
            BeamVec<DT>::open(global_get<vec4_t>(row.base + min(v, row.vecs - 1)), x);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int i = v * N + e - row.shift;
                const float y = beam_clean(x[e]);
                if (v < row.vecs && i >= 0 && i < row.vocab && y > -__builtin_inff()) f(comp_key(fkey(y + 0.0f), (uint32_t)i));
            }
        }
    };
    __syncthreads();
    if (tid == 0) S.count = 0;
    __syncthreads();
    int mine = 0;
    each([&](uint64_t) { ++mine; });
    atomicAdd(&S.count, mine);
    __syncthreads();
    const int need = min(most, S.count);
    __syncthreads();
    if (need == 0) return 0;
    constexpr int kShift[5] = {53, 42, 32, 10, 0}, kBits[5] = {11, 11, 10, 10, 10};
    uint64_t prefix = 0;
    int left = need;
#pragma unroll 1
    for (int p = 0; p < 5; ++p) {
        const int sh = kShift[p], bits = kBits[p], known = p == 3 ? 32 : sh + bits;     // bits 20..31 are the same in all
        if (p == 3) prefix |= 0xFFF00000u;
        for (int i = tid; i < 2048; i += kBeamThreads) S.hist[i] = 0;
        __syncthreads();
        const uint64_t want = known >= 64 ? 0 : prefix >> known;
        each([&](uint64_t c) {
            if ((known >= 64 ? 0 : c >> known) == want) atomicAdd(&S.hist[(uint32_t)(c >> sh) & ((1u << bits) - 1u)], 1u);
        });
        __syncthreads();
        // bins from the highest down: thread t sums 8 of them
        uint32_t own = 0;
        const int top = 2047 - 8 * tid;
#pragma unroll
        for (int i = 0; i < 8; ++i) own += S.hist[top - i];
        const uint32_t incl = wave_incl_scan_u32(own);
        if ((tid & 63) == 63) S.wave[tid >> 6] = incl;
        __syncthreads();
        uint32_t before = incl - own;
        for (int w = 0; w < (tid >> 6); ++w) before += S.wave[w];
        if (before < (uint32_t)left && before + own >= (uint32_t)left) {
            uint32_t sum = before;
            int b = top;
            while (sum + S.hist[b] < (uint32_t)left) sum += S.hist[b--];
            S.above = sum;
            S.bin = (uint32_t)b;
        }
        __syncthreads();
        left -= (int)S.above;
        prefix |= (uint64_t)S.bin << sh;
        __syncthreads();
    }
    if (tid == 0) S.count = 0;
    __syncthreads();
    each([&](uint64_t c) {
        if (c >= prefix) S.list[atomicAdd(&S.count, 1)] = c;
    });
    __syncthreads();
    return need;
}

// grid (spans, rows): a span's largest logit, its sum of exp, and its best candidates in order.
// One pass over the logits.  The first tile gives a bound: every wave finds what a quarter of the
// wanted candidates reach among its 64 lanes' maxima, and the least of the four waves' bounds is
// reached by all of them.  What reaches it is listed, in later tiles too; at the end the lists
// are cut by such a bound of their own and ranked.  Four instructions a logit and the exponential;
// 512 rows of 151936 in bf16 36 to 38 us (4.2 TB/s, a large copy has 4.9), 4 rows 6.8, 80 rows of 50001
// in fp32 8.3.
template <int DT>
__global__ __launch_bounds__(kBeamThreads, kBeamHold<DT>) void k_beam_scan(const fie_beam_args a, const BeamWork w)
{
    __shared__ BeamShared S;
    const int row_id = blockIdx.y, span = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (beam_dead(a, row_id)) return;
    const BeamRow<DT> row(a, row_id);
    constexpr int LOADS = BeamRow<DT>::LOADS;
    const int tiles = (row.vecs + LOADS * kBeamThreads - 1) / (LOADS * kBeamThreads);
    const int first = span * w.tiles, last = min(first + w.tiles, tiles);
    BeamSpan* out = w.span + (int64_t)row_id * w.spans + span;
    if (first >= last) {
        if (tid == 0) *out = BeamSpan{0.0, -kLargest, 0};
        return;
    }
    if (tid == 0) S.count = 0;
    uint64_t* const mine = S.list + wave * kBeamShare;
    int held = 0;
    const int rank = (w.most + kBeamWaves - 1) / kBeamWaves;
    float top = -kLargest, bound = -__builtin_inff();
    double sum = 0.0;
    vec4_t raw[LOADS];
    row.load(first, raw);
    for (int t = first; t < last; ++t) {
        float x[kBeamEach];
        row.open(t, raw, x);
        if (t + 1 < last) row.load(t + 1, raw);
        float part[4];                                  // maxima of eight logits each
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            part[g] = x[8 * g];
#pragma unroll
            for (int e = 1; e < 8; ++e) part[g] = __builtin_fmaxf(part[g], x[8 * g + e]);
        }
        float m = __builtin_fmaxf(__builtin_fmaxf(part[0], part[1]), __builtin_fmaxf(part[2], part[3]));
        float up = __builtin_fmaxf(top, m);
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < kBeamEach; ++e) s[e & 3] += __builtin_amdgcn_exp2f((x[e] - up) * kLog2e);
        float here = (s[0] + s[1]) + (s[2] + s[3]);
        if (__any(!(here == here) || up > kLargest)) {  // a NaN or an infinity among them
            m = -__builtin_inff();
#pragma unroll
            for (int e = 0; e < kBeamEach; ++e) {
                x[e] = beam_clean(x[e]);
                m = __builtin_fmaxf(m, x[e]);
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) part[g] = m;
            up = __builtin_fmaxf(top, m);
            here = 0.0f;
#pragma unroll
            for (int e = 0; e < kBeamEach; ++e) here += __builtin_amdgcn_exp2f((x[e] - up) * kLog2e);
        }
        if (up > top) sum *= __builtin_amdgcn_exp2f((top - up) * kLog2e);
        sum += here;
        top = up;
        if (t == first) {
            const uint32_t key = m > -__builtin_inff() ? fkey(m + 0.0f) : 0u;
            const uint32_t reach = beam_reach<16>(key, rank);
            if (lane == 0) S.wave[wave] = reach;
            __syncthreads();
            uint32_t least = S.wave[0];
#pragma unroll
            for (int i = 1; i < kBeamWaves; ++i) least = min(least, S.wave[i]);
            // a bound that some wave's lanes do not reach: everything is listed
            bound = least > kKeyNegInf ? key_to_float(least) : -kLargest;
        }
        // (places by ballot: with a counter in LDS a wave waited for it at each logit that was listed)
        if (__any(m >= bound))
#pragma unroll
            for (int g = 0; g < 4; ++g)
                if (__any(part[g] >= bound))
#pragma unroll
                    for (int e = 8 * g; e < 8 * g + 8; ++e) {
                        const uint64_t hits = __ballot(x[e] >= bound);
                        if (!hits) continue;
                        const int at = held + (int)__popcll(hits & ((1ull << lane) - 1ull));
                        if (x[e] >= bound && at < kBeamShare) mine[at] = comp_key(fkey(x[e] + 0.0f), (uint32_t)row.index(t, e));
                        held += (int)__popcll(hits);
                    }
    }
    // the span's maximum and sum
    float all = top;
    for (int d = 32; d; d >>= 1) all = __builtin_fmaxf(all, __shfl_xor(all, d, 64));
    if (lane == 0) S.top[wave] = all;
    __syncthreads();
    all = S.top[0];
#pragma unroll
    for (int i = 1; i < kBeamWaves; ++i) all = __builtin_fmaxf(all, S.top[i]);
    sum *= __builtin_amdgcn_exp2f((top - all) * kLog2e);
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d, 64);
    if (lane == 0) S.sum[wave] = sum;
    if (lane == 0) S.held[wave] = held;
    // a bound among what the waves listed, and what reaches it together
    uint64_t keep[kBeamShare / 64];
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i < kBeamShare / 64; ++i) {
        keep[i] = lane + i * 64 < held ? mine[lane + i * 64] : 0;
        best = max(best, comp_k(keep[i]));
    }
    const uint32_t reach = beam_reach<16>(best, rank);
    if (lane == 0) S.wave[wave] = reach;
    __syncthreads();
    uint32_t least = S.wave[0];
    bool over = false;
#pragma unroll
    for (int i = 0; i < kBeamWaves; ++i) {
        least = min(least, S.wave[i]);
        over |= S.held[i] > kBeamShare;
    }
#pragma unroll
    for (int i = 0; i < kBeamShare / 64; ++i)
        if (keep[i] && comp_k(keep[i]) >= least) S.list[atomicAdd(&S.count, 1)] = keep[i];
    __syncthreads();
    int count = over ? kBeamList + 1 : S.count;
    if (count > 2 * kBeamThreads) count = beam_deep<DT>(row, first, last, w.most, S);
    // each entry's place
    uint64_t* cand = w.cand + ((int64_t)row_id * w.spans + span) * w.most;
    for (int i = tid; i < count; i += kBeamThreads) {
        const uint64_t c = S.list[i];
        int place = 0;
        for (int j = 0; j < count; ++j) place += S.list[j] > c;
        if (place < w.most) cand[place] = c;
    }
    if (tid == 0) *out = BeamSpan{(S.sum[0] + S.sum[1]) + (S.sum[2] + S.sum[3]), all, min(count, w.most)};
}

// The order of doubles as that of whole numbers; -inf and NaN are 0, no continuation.
FIE_DEV uint64_t beam_order(double v)
{
    if (!(v > -__builtin_inf())) return 0;
    const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
    return b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
}

FIE_DEV double beam_value(uint64_t k)
{
    return __longlong_as_double((int64_t)((k >> 63) ? (k & 0x7FFFFFFFFFFFFFFFull) : ~k));
}

// A score or an answer's value: none is -inf, which says that nothing is there.
FIE_DEV float beam_held(double v) { return __builtin_fmaxf((float)v, -kLargest); }

// length^penalty.  (The exponential and the logarithm as they are shared with a row's: a power's own code
// takes longer to come in than to run.)
__host__ FIE_DEV bool beam_power(double penalty) { return penalty != 0.0 && penalty != 1.0; }
FIE_DEV double beam_scale(int length, double penalty)
{
    if (penalty == 1.0) return (double)length;
    if (penalty == 0.0) return 1.0;
    return exp(penalty * log((double)length));
}

// An answer's value.  (A power out of a double's range is 0 or an infinity: no total but 0 is left
// undefined by that, and it is 0 at any length.)
FIE_DEV float beam_ended(double total, double scale) { return total != 0.0 ? beam_held(total / scale) : 0.0f; }

// What a request's workgroup settles before the pool.
struct BeamChoice {
    double lse[FIE_MAX_BEAMS];                          // log of a row's sum, less its maximum
    double scale;                                       // of an answer that ends here
    float top[FIE_MAX_BEAMS], prior[FIE_MAX_BEAMS];
    int32_t count[FIE_MAX_BEAMS];
    uint64_t live_key[FIE_MAX_BEAMS];
    int32_t live_token[FIE_MAX_BEAMS], live_beam[FIE_MAX_BEAMS];
    float end_value[FIE_MAX_BEAMS];
    int32_t end_token[FIE_MAX_BEAMS], end_beam[FIE_MAX_BEAMS];
    int32_t found, ended, listed;
    uint32_t wave[16];
};

// The order of a beam's continuation by a token of logit x.  (In fp32 x - top would be off by 2^-24 of
// it: tokens far below the top would tie across beams.)
FIE_DEV uint64_t beam_total(const BeamChoice& C, int beam, float x)
{
    return beam_order((double)C.prior[beam] + (((double)x - (double)C.top[beam]) - C.lse[beam]));
}

constexpr int kPickEach = 4;                            // candidates of a thread
constexpr int kPickList = 1024;                         // those that are ranked

// A thread's n-th candidate: the waves take turns, another first each time, so that each has its share of
// the good beams' and of the lists' heads (a wave of bad beams alone, or of each list's last
// alone where as many are listed as there are waves, lowers the bound to all there are: 20 us for 10).
FIE_DEV int pick_index(int n)
{
    const int waves = blockDim.x >> 6, turn = (threadIdx.x & 63) + 64 * n;
    return turn * waves + ((threadIdx.x >> 6) + turn) % waves;
}

FIE_DEV bool is_eos(const fie_beam_args& a, int token)
{
    bool eos = false;
    for (int i = 0; i < a.eos_count; ++i) eos |= token == a.eos[i];
    return eos;
}

// A continuation in the request's order: `first` by its total, `then` on ties, by the lower beam, the
// larger logit and the lower token (of 20 bits).
FIE_DEV uint64_t pick_then(int beam, uint64_t cand)
{
    return ((uint64_t)(63 - beam) << 52) | ((uint64_t)comp_k(cand) << 20) | ((uint32_t)cand & 0xFFFFFu);
}
FIE_DEV int then_beam(uint64_t t) { return 63 - (int)(t >> 52); }
FIE_DEV int then_token(uint64_t t) { return 0xFFFFF - (int)(t & 0xFFFFFu); }

// All of a request's candidates at once: a bound on their totals as in the scan, what reaches it into a
// list, the list by rank, and its places in order by a wave's ballots.  False where more reach it than
// the list holds (many equal totals).  `wanted`: as many as may stand in front of the last that goes on.
FIE_DEV bool pick_ranked(const fie_beam_args& a, const BeamWork& w, int r, int wanted, int length, double scale, uint64_t* L,
                         const uint64_t (&cand)[kPickEach], BeamChoice& C)
{
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
    const int per = w.spans * w.most, all = a.beams * per;
    uint64_t key[kPickEach];
    uint32_t best = 0;
#pragma unroll
    for (int n = 0; n < kPickEach; ++n) {
        const int i = pick_index(n), beam = i < all ? i / per : 0;
        key[n] = 0;
        if (cand[n]) key[n] = beam_total(C, beam, key_to_float(comp_k(cand[n])));
        best = max(best, (uint32_t)(key[n] >> 32));
    }
    const uint32_t reach = beam_reach<4>(best, (wanted + waves - 1) / waves);
    if (lane == 0) C.wave[wave] = reach;
    __syncthreads();
    uint32_t least = C.wave[0];
    for (int i = 1; i < waves; ++i) least = min(least, C.wave[i]);
    uint64_t* const first = L;
    uint64_t* const then = L + kPickList;
#pragma unroll
    for (int n = 0; n < kPickEach; ++n)
        if (key[n] && (uint32_t)(key[n] >> 32) >= least) {
            const int at = atomicAdd(&C.listed, 1), i = pick_index(n);
            if (at < kPickList) {
                first[at] = key[n];
                then[at] = pick_then(i / per, cand[n]);
            }
        }
    __syncthreads();
    const int count = C.listed;
    if (count > kPickList) return false;
    uint64_t* const first_s = then + kPickList;         // in order
    uint64_t* const then_s = first_s + kPickList;
#pragma unroll 1
    for (int i = tid; i < count; i += blockDim.x) {
        const uint64_t f = first[i], t = then[i];
        int place = 0;
#pragma unroll 8
        for (int j = 0; j < count; ++j) place += first[j] > f || (first[j] == f && then[j] > t);
        first_s[place] = f;
        then_s[place] = t;
    }
    __syncthreads();
    if (wave) return true;
    const bool last = a.max_tokens > 0 && length + 1 >= a.max_tokens;           // all end
    const uint64_t below = (1ull << lane) - 1ull;
    int live = 0, ends = 0, rank = 0;
#pragma unroll 1
    for (int i0 = 0; i0 < count && live < a.beams && !(last && rank >= a.beams); i0 += 64) {
        const int i = i0 + lane;
        const uint64_t f = i < count ? first_s[i] : 0, t = i < count ? then_s[i] : 0;
        const int token = then_token(t);
        const bool eos = f && is_eos(a, token), exists = f && !(eos && length + 1 < a.min_tokens), goes = exists && !eos && !last;
        const uint64_t any = __ballot(exists), on = __ballot(goes);
        const int my_rank = rank + (int)__popcll(any & below), my_live = live + (int)__popcll(on & below);
        const bool stops = exists && !goes && my_rank < a.beams;
        const uint64_t off = __ballot(stops);
        if (goes && my_live < a.beams) {
            C.live_key[my_live] = f;
            C.live_token[my_live] = token;
            C.live_beam[my_live] = then_beam(t);
        }
        if (stops) {
            const int at = ends + (int)__popcll(off & below);
            C.end_value[at] = beam_ended(beam_value(f), scale);
            C.end_token[at] = token;
            C.end_beam[at] = then_beam(t);
        }
        rank += (int)__popcll(any);
        live += (int)__popcll(on);
        ends += (int)__popcll(off);
    }
    if (lane == 0) {
        C.found = min(live, a.beams);
        C.ended = ends;
    }
    return true;
}

// The same one by one, for any number: a wave a row at first, whose spans' lists are in order, so that
// its best candidates come off their heads; then the request's, off its rows' lists, in one wave
// with a beam a lane.  A few hundred cycles a candidate.  LDS: [waves][spans][most], [beams][most].
FIE_DEV void pick_one_by_one(const fie_beam_args& a, const BeamWork& w, int r, int length, double scale, uint64_t* L, BeamChoice& C)
{
    const int K = a.beams, lane = threadIdx.x & 63, most = w.most;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    uint64_t* heads = L + (int64_t)wave * w.spans * most;
    uint64_t* rows = L + (int64_t)waves * w.spans * most;
#pragma unroll 1
    for (int b = wave; b < K; b += waves) {
        if (C.count[b] == 0) continue;
        const int64_t row = (int64_t)r * K + b;
        const int held = lane < w.spans ? w.span[row * w.spans + lane].count : 0;
        const uint64_t* from = w.cand + row * w.spans * most;
        for (int i = lane; i < w.spans * most; i += 64) heads[i] = from[i];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        int at = 0, n = 0;
        uint64_t head = held > 0 ? heads[lane * most] : 0;
#pragma unroll 1
        for (; n < most; ++n) {
            const uint64_t best = dwave_max_u64(head);
            if (best == 0) break;
            if (lane == 0) rows[b * most + n] = best;
            if (head == best) {
                ++at;
                head = at < held ? heads[lane * most + at] : 0;
            }
        }
        if (lane == 0) C.count[b] = n;
    }
    __syncthreads();
    if (wave) return;
    const int n = lane < K ? C.count[lane] : 0;
    int at = 0;
    auto look = [&]() {
        if (at >= n) return (uint64_t)0;
        return beam_total(C, lane, key_to_float(comp_k(rows[lane * most + at])));
    };
    uint64_t head = look();
    int live = 0, ends = 0, rank = 0;
    const bool last = a.max_tokens > 0 && length + 1 >= a.max_tokens;           // all end
#pragma unroll 1
    while (live < K && !(last && rank >= K)) {
        const uint64_t best = dwave_max_u64(head);
        if (best == 0) break;
        const int who = (int)__builtin_ctzll(__ballot(head == best));           // ties: the lower beam
        const int token = (int)comp_idx(rows[who * most + __builtin_amdgcn_readlane(at, who)]);
        bool eos = is_eos(a, token);
        if (lane == who) {
            ++at;
            head = look();
        }
        if (eos && length + 1 < a.min_tokens) continue;                         // does not exist
        eos |= last;
        if (lane == 0) {
            if (!eos) {
                C.live_key[live] = best;
                C.live_token[live] = token;
                C.live_beam[live] = who;
            } else if (rank < K) {
                C.end_value[ends] = beam_ended(beam_value(best), scale);
                C.end_token[ends] = token;
                C.end_beam[ends] = who;
            }
        }
        if (!eos) ++live;
        else if (rank < K) ++ends;
        ++rank;
    }
    if (lane == 0) {
        C.found = live;
        C.ended = ends;
    }
}

// A workgroup a request: its rows' logarithms, a wave each, then its best continuations, then the pool.
// Bound by the chain of these steps, and by how much code each of them has to bring in: 1 request of 4
// beams 9 us, 64 of 8 beams 11 (one candidate after the other 9 and 14); one by one for a request of 64
// beams at 50257 166.
__global__ __launch_bounds__(1024) void k_beam_pick(const fie_beam_args a, const BeamWork w, int wanted)
{
    extern __shared__ uint64_t L[];
    __shared__ BeamChoice C;
    __shared__ float old_value[FIE_MAX_BEAMS];
    __shared__ int32_t old_end[FIE_MAX_BEAMS][3];
    const int r = blockIdx.x, K = a.beams, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = blockDim.x >> 6;
    const int per = w.spans * w.most;
    // every load at once: what a row that is not there left in the workspace is looked at by no one
    uint64_t cand[kPickEach];
    int32_t held[kPickEach];
    if (wanted)
#pragma unroll
        for (int n = 0; n < kPickEach; ++n) {
            const int i = pick_index(n), at = min(i, K * per - 1), list = at / w.most;
            cand[n] = w.cand[(int64_t)r * K * per + at];
            held[n] = i < K * per ? w.span[(int64_t)r * K * w.spans + list].count - (at - list * w.most) : 0;
        }
    const int length = a.lengths[r];
    const bool was = a.done[r] != 0;
    if (tid < K) {
        const float p = a.pool[r * K + tid], s = a.scores[r * K + tid];
        old_value[tid] = p == p ? p : -__builtin_inff();
        for (int i = 0; i < 3; ++i) old_end[tid][i] = a.ends[(r * K + tid) * 3 + i];
        C.prior[tid] = s;
        C.count[tid] = !was && s > -__builtin_inff();
    }
    if (tid == 0) C.listed = 0;
    __syncthreads();
    const int workers = beam_power(a.length_penalty) ? waves - 1 : waves;       // (the last wave has the length's power)
#pragma unroll 1
    for (int b = wave; b < K; b += workers) {
        if (wave >= workers || C.count[b] == 0) continue;
        const BeamSpan sp = lane < w.spans ? w.span[((int64_t)r * K + b) * w.spans + lane] : BeamSpan{0.0, -kLargest, 0};
        float m = sp.top;
        for (int d = 32; d; d >>= 1) m = __builtin_fmaxf(m, __shfl_xor(m, d, 64));
        double s = sp.sum * __builtin_amdgcn_exp2f((sp.top - m) * kLog2e);
        for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d, 64);
        if (lane == 0) {
            C.top[b] = m;
            C.lse[b] = log(s);
        }
    }
    if (wave == waves - 1) {                            // (where it is none, at no cost)
        const double scale = beam_scale(max(was ? length : length + 1, 1), a.length_penalty);
        if (lane == 0) C.scale = scale;
    }
    __syncthreads();
    const double scale = C.scale;
    bool ranked = wanted > 0;
    if (ranked) {
#pragma unroll
        for (int n = 0; n < kPickEach; ++n) {
            const int i = pick_index(n);
            if (held[n] <= 0 || C.count[min(i / per, K - 1)] == 0) cand[n] = 0;
        }
        ranked = pick_ranked(a, w, r, wanted, length, scale, L, cand, C);
    }
    if (!ranked) {
        __syncthreads();
        pick_one_by_one(a, w, r, length, scale, L, C);
    }
    __syncthreads();
    if (wave) return;
    // the pool: its own and the new ones by value, the older first; both are held before the writes
    const int E = C.ended, live = C.found;
    const float mine = lane < K ? old_value[lane] : -__builtin_inff();
    int place = 64;
    if (lane < K) {
        place = 0;
        for (int j = 0; j < K; ++j) place += old_value[j] > mine || (old_value[j] == mine && j < lane);
        for (int j = 0; j < E; ++j) place += C.end_value[j] > mine;
    }
    int fresh = 64;
    if (lane < E) {
        fresh = 0;
        const float v = C.end_value[lane];
        for (int j = 0; j < K; ++j) fresh += old_value[j] >= v;
        for (int j = 0; j < E; ++j) fresh += C.end_value[j] > v || (C.end_value[j] == v && j < lane);
    }
    auto put = [&](int to, float v, int e0, int e1, int e2) {
        a.next_pool[r * K + to] = v;
        int32_t* e = a.next_ends + (int64_t)(r * K + to) * 3;
        e[0] = e0;
        e[1] = e1;
        e[2] = e2;
    };
    if (place < K) put(place, mine, old_end[lane][0], old_end[lane][1], old_end[lane][2]);
    if (fresh < K) put(fresh, C.end_value[lane], length + 1, r * K + C.end_beam[lane], C.end_token[lane]);
    // the pool's worst
    float worst = __builtin_inff();
    if (place == K - 1) worst = mine;
    if (fresh == K - 1) worst = C.end_value[lane];
    for (int d = 32; d; d >>= 1) worst = __builtin_fminf(worst, __shfl_xor(worst, d, 64));
    bool done = was || live == 0;
    if (!done && worst > -__builtin_inff()) done = a.early_stopping || worst >= beam_ended(beam_value(C.live_key[0]), scale);
    if (lane < K) {
        const int row = r * K + lane;
        const bool goes = !done && lane < live;
        const int token = goes ? C.live_token[lane] : a.pad, parent = goes ? r * K + C.live_beam[lane] : row;
        a.next_scores[row] = goes ? beam_held(beam_value(C.live_key[lane])) : -__builtin_inff();
        a.tokens[row] = token;
        a.parents[row] = parent;
        if (a.history_tokens && !was && length >= 0 && length < a.history_steps) {
            const int64_t to = (int64_t)length * a.requests * K + row;
            a.history_tokens[to] = token;
            a.history_parents[to] = parent;
        }
    }
    if (lane == 0) {
        a.next_lengths[r] = was ? length : length + 1;
        a.next_done[r] = done;
    }
}

}  // namespace fie
