// Verification of drafted tokens behind the sampler's kernels (fie_sampler_verify).
//
// k_accept tests a request's drafts: p(d_j) from the row's thresholds, tile maxima and kept
// mass, which the sampler left in the workspace.  k_refused draws the token of a refusal from
// what the row's p has over the draft's q, over one row of logits and one of q a request: spans
// sum the excess as whole numbers (fixed point, 2^-48: sums have no order), and the last span
// of a request to arrive finds the tile and the token the draw lands in.
#pragma once

#include "launchers.h"

namespace fie {

constexpr int kVerThreads = 256;
constexpr int kVerTiles = 4;               // tiles a workgroup of k_refused and k_rank, or one

// A draw that k_accept leaves for k_refused: all that its workgroups need, in one place (they
// are a chain of dependent loads otherwise: 2 refusals took 16-22 us, the draws themselves 8).
struct VerJob {
    double total;       // the row's kept mass
    double u;
    int64_t draft;      // the refused draft, of all drafts
    int64_t id;
    int64_t* out;       // where the token goes
    int32_t row;        // -1: nothing to draw
    int32_t lim;        // a refusal's; kRankDraw: a draw of the row in rank order instead
    float edge, s;      // edge: a rank draw's bins a unit
};
constexpr int kRankDraw = -1;

// In workspace arrays that the sampler is done with.
struct VerWs {
    VerJob* job;        // [requests]
    uint32_t* arrived;  // [requests]
    uint64_t* sum;      // [requests * tiles]
};
static_assert(sizeof(VerJob) <= sizeof(DeferRec), "jobs go where the deferred rows' records were");

// What of a row is kept: tokens above `edge`, and those at it up to token `lim`.  (The sampler's
// rule is key >= tau and (key, index) >= cut in rank order; the later of the two decides.)
struct Kept {
    float edge;
    int lim;
    FIE_DEV Kept(float e, int l) : edge(e), lim(l) {}
    FIE_DEV explicit Kept(const RowRes& rr)
    {
        const uint32_t ck = comp_k(rr.cut);
        const bool at_cut = rr.cut != 0 && ck >= rr.tau;
        const uint32_t k = at_cut ? ck : rr.tau;
        edge = k > kKeyNegInf ? key_to_float(k) : -__builtin_inff();
        lim = at_cut ? (int)comp_idx(rr.cut) : 0x7FFFFFFF;
    }
    FIE_DEV bool operator()(float y, int idx) const { return y > edge || (y == edge && idx <= lim); }
    FIE_DEV bool all() const { return edge == -__builtin_inff() && lim == 0x7FFFFFFF; }
};

FIE_DEV double mass_of(const RowRes& rr) { return u128_to_double(((u128)rr.khi << 64) | rr.klo); }

// A tile's share of the kept mass per unit of weight.
FIE_DEV float share_of(uint64_t ct, double total) { return total > 0.0 ? (float)((double)ct / total) : 0.0f; }

// A kept token's probability: its weight (below 2^41; weight20 2^20, floored) by the share.
FIE_DEV float prob_of(float y, float m, float share) { return __builtin_floorf(weight20(y - m) * 0x1p20f) * share; }

FIE_DEV float row_scale(float x, float s) { return s == 1.0f ? x + 0.0f : scaled(x, s); }

// The request's drafts and rows; false where its offsets do not fit.
struct Request {
    int64_t first;      // of its drafts
    int k, row;         // drafts, first row
};
FIE_DEV bool request_of(const KParams& P, const fie_verify_args& v, int r, Request* q)
{
    const int64_t a = v.draft_offsets[r], b = v.draft_offsets[r + 1];
    const int64_t drafts = (int64_t)P.a.rows - v.requests;
    if (a < 0 || b < a || b - a > v.max_drafts || b > drafts) return false;
    q->first = a;
    q->k = (int)(b - a);
    q->row = (int)(a + r);
    return true;
}

// A draft's probability as fp32, at least 0 (NaN: 0).
FIE_DEV float at_least_0(float q) { return q > 0.0f ? q : 0.0f; }

FIE_DEV float draft_prob(const fie_verify_args& v, int64_t draft, int64_t id)
{
    const size_t o = (size_t)draft * (size_t)v.draft_stride + (size_t)id;
    if (v.draft_dtype == FIE_F32) return at_least_0(((const float*)v.draft_probs)[o]);
    const uint32_t h = ((const uint16_t*)v.draft_probs)[o];
    return at_least_0(v.draft_dtype == FIE_F16 ? lane_get<FIE_F16>(make_uint4(h, 0, 0, 0), 0)
                                               : lane_get<FIE_BF16>(make_uint4(h, 0, 0, 0), 0));
}

FIE_DEV uint32_t history_count(const fie_sampler_args& a, int row, uint32_t id, int lane)
{
    const int64_t h1 = hist_end(a, row);
    uint32_t n = 0;
    for (int64_t h = a.hist_offsets[row] + lane; h < h1; h += 64) n += (uint32_t)a.hist_ids[h] == id;
    return dwave_sum_u32(n);
}

// A row as the kernels that go over it by spans see it.
template <int DT, int TPS_>
struct SpanRow {
    static constexpr int EPL = DTy<DT>::EPL, TPS = TPS_, kSpanV = TPS * kTile;     // tiles, tokens a span
    static constexpr int GPT = kTile / (kVerThreads * EPL);         // groups of the workgroup a tile
    static constexpr int NL = TPS * GPT;                            // ... a span
    const KParams& P;
    int row;
    bool pen, quick;
    float rep, pres, freq, s, rs;
    const char* rowp;
    const float* mt;        // the tiles' largest scaled logits, token 0's first
    const uint64_t* ct;     // their scales
    float m0;
    uint32_t* cnt;          // the workgroup's LDS: a span's penalty counts

    FIE_DEV SpanRow(const KParams& P_, int row_, float s_, uint32_t* cnt_) : P(P_), row(row_), s(s_), cnt(cnt_)
    {
        const fie_sampler_args& a = P.a;
        mt = P.w.mt + (size_t)row * (P.NT + 1);
        ct = P.w.ct + (size_t)row * (P.NT + 1);
        m0 = mt[0];
        pen = a.apply_penalties && (a.flags[row] & FIE_FLAG_PENALTY);
        rep = pen ? a.repetition[row] : 1.0f;
        pres = pen ? a.presence[row] : 0.0f;
        freq = pen ? a.frequency[row] : 0.0f;
        rowp = (const char*)a.logits + (size_t)row * (size_t)a.row_stride * DTy<DT>::SZ;
        // the divide by Markstein's correction where it is exact, and where neither answer
        // counts (an infinite logit's weight is 0 either way)
        rs = 1.0f / s;
        quick = s >= 0x1p-30f && s <= 0x1p30f;
    }
    FIE_DEV uint4 load(int e0) const { return load_group<DT>(rowp, e0, P.a.vocab); }

    FIE_DEV void count(int lo) const
    {
        const fie_sampler_args& a = P.a;
        __syncthreads();
        for (int i = threadIdx.x; i < kSpanV; i += kVerThreads) cnt[i] = 0;
        __syncthreads();
        const int64_t h1 = hist_end(a, row);
        for (int64_t h = a.hist_offsets[row] + threadIdx.x; h < h1; h += kVerThreads) {
            const uint32_t id = (uint32_t)a.hist_ids[h];
            if (id >= (uint32_t)lo && id - (uint32_t)lo < (uint32_t)kSpanV && id < (uint32_t)a.vocab) atomicAdd(&cnt[id - lo], 1u);
        }
        __syncthreads();
    }
    // The scaled logits of the EPL tokens from e0 on, as loaded, of the span (or tile) from lo
    // on that was counted last.
    FIE_DEV void values(int lo, int e0, const uint4& raw, float (&y)[EPL]) const
    {
        bool odd = false;
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
            float x = lane_get<DT>(raw, e);
            if (pen && e0 + e < P.a.vocab && cnt[e0 + e - lo]) x = penalize(x, rep, pres, freq, cnt[e0 + e - lo]);
            const float ax = __builtin_fabsf(x);
            odd |= (DT != FIE_F16 || pen) && ((ax < 0x1p-96f && ax > 0.0f) || (ax > 0x1p96f && ax < __builtin_inff()));
            y[e] = x;
        }
        if (s == 1.0f) {
#pragma unroll
            for (int e = 0; e < EPL; ++e) y[e] += 0.0f;
        } else if (quick && __ballot(odd) == 0) {
#pragma unroll
            for (int e = 0; e < EPL; ++e) y[e] = div_markstein(y[e], s, rs) + 0.0f;
        } else {
#pragma unroll
            for (int e = 0; e < EPL; ++e) y[e] = scaled(y[e], s);
        }
        if (e0 == 0) y[0] = m0;             // token 0 is a tile of its own
    }
};

// After its own stores and atomics at device scope, a workgroup counts itself in; true in every
// thread of the last of `all`.
FIE_DEV bool arrive_last(uint32_t* count, uint32_t all, uint32_t* flag)
{
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0)
        *flag = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == all - 1;
    __syncthreads();
    return *flag != 0;
}

template <typename T> FIE_DEV T from_all(const T* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename T> FIE_DEV void to_all(T* p, T v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

}  // namespace fie

#include "verify_draw.h"

namespace fie {

// One workgroup a request: draft j by thread j; on rows with penalties the draft's
// occurrences in the row's history are counted first, a wave a draft.
//
// A draft's p from one logit and its tile's maximum and scale: the row is not read again, so
// the kernel is a chain of three dependent loads (offsets, draft, logit and tile) whatever the
// vocabulary: 4.7 us for 1 request of 4 drafts, 7.3 for 256 (rank_begin's bins among them).
template <int DT>
__global__ __launch_bounds__(kVerThreads) void k_accept(const KParams P, const fie_verify_args v, const VerWs vw)
{
    __shared__ uint32_t cnt[FIE_MAX_DRAFTS + 1];
    __shared__ uint32_t red[kVerThreads / 64];
    const fie_sampler_args& a = P.a;
    const int r = blockIdx.x, tid = threadIdx.x, V = a.vocab;
    int64_t* out = v.tokens + (size_t)r * (v.max_drafts + 1);
    Request q;
    if (!request_of(P, v, r, &q)) {                            // the same in every thread
        for (int j = tid; j <= v.max_drafts; j += kVerThreads) out[j] = -1;
        if (tid == 0) { v.accepted[r] = -1; vw.job[r].row = -1; }
        return;
    }
    if (a.apply_penalties) {
        for (int j = tid >> 6; j < q.k; j += kVerThreads / 64) {
            const int row = q.row + j;
            const int64_t d = v.draft_ids[q.first + j];
            const bool count = (a.flags[row] & FIE_FLAG_PENALTY) && d > 0 && d < V;
            const uint32_t n = count ? history_count(a, row, (uint32_t)d, tid & 63) : 0;
            if ((tid & 63) == 0) cnt[j] = n;
        }
        __syncthreads();
    }
    uint32_t refused = 0xFFFFFFFFu;
    int64_t id = -1;
    if (tid < q.k) {
        const int row = q.row + tid;
        const int32_t fl = a.flags[row];
        id = v.draft_ids[q.first + tid];
        float p = 0.0f, qd = 0.0f;
        if (id >= 0 && id < V) {
            const RowRes rr = P.w.res[row];
            const size_t slot = (size_t)row * (P.NT + 1) + (id ? 1 + (int)id / kTile : 0);
            const float m = P.w.mt[slot];
            const uint64_t ct = P.w.ct[slot];
            const char* rowp = (const char*)a.logits + (size_t)row * (size_t)a.row_stride * DTy<DT>::SZ;
            float x = load_elem<DT>(rowp, (uint32_t)id);
            qd = v.draft_probs ? draft_prob(v, q.first + tid, id) : 1.0f;
            if (rr.greedy) {
                p = id == rr.token ? 1.0f : 0.0f;
            } else {
                if (a.apply_penalties && cnt[tid]) x = penalize(x, a.repetition[row], a.presence[row], a.frequency[row], cnt[tid]);
                const float y = id ? row_scale(x, rr.s) : m;        // token 0 is a tile of its own
                p = Kept(rr)(y, (int)id) ? prob_of(y, m, share_of(ct, mass_of(rr))) : 0.0f;
            }
        }
        if (v.target_probs) v.target_probs[q.first + tid] = p;
        const double u = row_uniform(a, row, fl & ~FIE_FLAG_NO_DRAW);
        if (!(u * (double)qd < (double)p)) refused = (uint32_t)tid;
    }
    const int n = (int)min(block_min_u32<kVerThreads>(refused, red), (uint32_t)q.k);
    if (tid < n) out[tid] = id;
    if (tid > n && tid <= v.max_drafts) out[tid] = -1;
    // A request that keeps every draft and whose last row carries FIE_FLAG_NO_DRAW is drawn from
    // by the passes of verify_draw.h.
    const int end = q.row + q.k;
    const bool rank = v.draws && n == q.k && mass_only(a, end, a.flags[end]);
    if (rank) rank_begin(P, end, red);
    if (tid == 0) {
        v.accepted[r] = n;
        vw.arrived[r] = 0;
        // no draw left: every draft kept (and the last row drawn from), or a greedy row
        const RowRes rr = P.w.res[q.row + n];
        const bool none = rank ? (rr.klo | rr.khi) == 0 : n == q.k || rr.greedy;
        VerJob job{};
        job.row = -1;
        if (none) {
            out[n] = a.tokens[q.row + n];
        } else {
            const Kept kept(rr);
            job.total = mass_of(rr);
            job.u = row_uniform(a, end, a.flags[end] & ~FIE_FLAG_NO_DRAW);
            job.out = out + n;
            job.row = q.row + n;
            job.s = rr.s;
            if (rank) {
                job.lim = kRankDraw;
            } else {
                job.draft = q.first + n;
                job.id = v.draft_ids[job.draft];
                job.lim = kept.lim;
                job.edge = kept.edge;
            }
        }
        vw.job[r] = job;
    }
}

// N tokens of a row of draft probabilities from e0 on, as loaded; past V: 0.
template <int QT, int N>
struct DraftVec {
    static constexpr int EPL = QT >= 0 ? DTy<QT < 0 ? 0 : QT>::EPL : N, G = N > EPL ? N / EPL : 1;
    uint4 w[G];
    FIE_DEV void load(const char* rowp, int e0, int V)
    {
        if constexpr (N >= EPL) {
#pragma unroll
            for (int g = 0; g < G; ++g) w[g] = load_group<QT>(rowp, e0 + g * EPL, V);
        } else {            // four of eight 16-bit values
            const uint16_t* p = (const uint16_t*)rowp + e0;
            uint32_t h[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = e0 + e < V ? p[e] : 0u;
            w[0] = make_uint4(h[0] | (h[1] << 16), h[2] | (h[3] << 16), 0, 0);
        }
    }
    FIE_DEV float get(int e) const { return at_least_0(lane_get<QT < 0 ? 0 : QT>(w[N >= EPL ? e / EPL : 0], N >= EPL ? e % EPL : e)); }
};

// What is left of a token, 2^-48 a unit, as two 24-bit parts: sums of 32 of each stay in 32 bits.
struct Excess { uint32_t hi, lo; };
FIE_DEV Excess excess_of(float p, float q)
{
    const float t = __builtin_fmaxf(p - q, 0.0f) * 0x1p24f;        // NaN: 0
    return Excess{(uint32_t)t, (uint32_t)(__builtin_amdgcn_fractf(t) * 0x1p24f)};
}

// Grid (spans, requests).  QT: the draft's type, -1 without probabilities.
//
// Bound by the two rows' way from memory, so what the sampler's tile maxima rule out is not
// read: a tile whose largest logit is below the row's edge, and q of a wave's tokens when none
// of them is kept.  A span a workgroup, since a refusal's row and its q (0.9 MB at vocab 151936)
// are far too much for one CU's loads.  256 requests of
// 4 drafts, bf16 logits and fp32 q: 39 us, 133 refusals and the first pass of 123 rank draws,
// 158 MB at most, 4 TB/s.  Few requests wait on the loads and on the last span's second look:
// 16 without q 16 us.
template <int DT, int QT, int TPS>
__global__ __launch_bounds__(kVerThreads) void k_refused(const KParams P, const fie_verify_args v, const VerWs vw)
{
    constexpr int EPL = DTy<DT>::EPL, SZ = DTy<DT>::SZ, NL = TPS * kTile / kVerThreads / EPL;
    extern __shared__ uint32_t cnt[];       // a span's, with penalties
    constexpr int WV = kVerThreads / 64;
    __shared__ uint64_t red[WV], tile_part[TPS][WV];
    __shared__ uint64_t left;
    __shared__ uint32_t found, last;
    const fie_sampler_args& a = P.a;
    const int r = blockIdx.y, tid = threadIdx.x, V = a.vocab, spans = gridDim.x;
    const VerJob J = vw.job[r];
    if (J.row < 0) return;
    if (J.lim == kRankDraw) {
        rank_pass<DT, 1, TPS>(P, vw, r, J, cnt);
        return;
    }
    const int row = J.row;
    const Kept kept(J.edge, J.lim);
    const SpanRow<DT, TPS> R(P, row, J.s, cnt);
    const char* qp = nullptr;
    if constexpr (QT >= 0) qp = (const char*)v.draft_probs + (size_t)J.draft * (size_t)v.draft_stride * DTy<QT>::SZ;
    const bool all = kept.all();            // no filter

    // a span's tiles: their largest scaled logits and their shares
    constexpr int GPT = SpanRow<DT, TPS>::GPT, kSpanV = TPS * kTile;
    struct Tiles { float m[TPS], share[TPS]; };
    auto tiles_of = [&](int lo) {
        Tiles t;
        uint64_t c[TPS];
#pragma unroll
        for (int i = 0; i < TPS; ++i) {
            const int slot = min(1 + lo / kTile + i, P.NT);
            t.m[i] = R.mt[slot];
            c[i] = R.ct[slot];
        }
#pragma unroll
        for (int i = 0; i < TPS; ++i) t.share[i] = share_of(c[i], J.total);
        return t;
    };
    const float m0 = R.m0;
    const uint64_t c0 = R.ct[0];
    // what p has over q at the EPL tokens from e0 on, in a tile with maximum m, from the logits
    // as loaded
    auto excess = [&](int lo, int e0, float m, float sh, uint4 raw, DraftVec<QT, EPL> dv, bool have_q, Excess (&w)[EPL]) {
        float y[EPL];
        bool any = false;
        R.values(lo, e0, raw, y);
#pragma unroll
        for (int e = 0; e < EPL; ++e) any |= kept(y[e], e0 + e);
        if (__ballot(any) == 0) {
#pragma unroll
            for (int e = 0; e < EPL; ++e) w[e] = Excess{0, 0};
            return;
        }
        if constexpr (QT >= 0)
            if (!have_q) dv.load(qp, e0, V);
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
            const int idx = e0 + e;
            float p = prob_of(y[e], m, sh);
            if (idx == 0) p = prob_of(m0, m0, share_of(c0, J.total));
            if (!kept(y[e], idx)) p = 0.0f;
            float qv;
            if constexpr (QT >= 0) qv = dv.get(e);
            else qv = idx == J.id ? 1.0f : 0.0f;
            w[e] = excess_of(idx < V ? p : 0.0f, qv);
        }
    };

    const int lo = blockIdx.x * kSpanV;
    if (R.pen) R.count(lo);
    {
        const Tiles t = tiles_of(lo);
        // a tile all below the edge holds nothing (token 0's own tile aside)
        auto skip = [&](int i) { return lo + i * kTile >= V || (t.m[i] < kept.edge && lo + i * kTile != 0); };
        uint4 raw[NL];
        DraftVec<QT, EPL> qs[NL];
#pragma unroll
        for (int j = 0; j < NL; ++j) {
            const int e0 = lo + (j * kVerThreads + tid) * EPL;
            raw[j] = make_uint4(0, 0, 0, 0);
            if (!skip(j / GPT)) {
                raw[j] = R.load(e0);
                if constexpr (QT >= 0)
                    if (all) qs[j].load(qp, e0, V);
            }
        }
#pragma unroll
        for (int i = 0; i < TPS; ++i) {
            uint64_t part = 0;
            if (!skip(i)) {
                uint32_t hi = 0, lw = 0;
#pragma unroll
                for (int j = i * GPT; j < (i + 1) * GPT; ++j) {
                    Excess w[EPL];
                    excess(lo, lo + (j * kVerThreads + tid) * EPL, t.m[i], t.share[i], raw[j], qs[j], all, w);
#pragma unroll
                    for (int e = 0; e < EPL; ++e) { hi += w[e].hi; lw += w[e].lo; }
                }
                part = dwave_sum_u64(((uint64_t)hi << 24) + lw);
            }
            if ((tid & 63) == 0) tile_part[i][tid >> 6] = part;
        }
    }
    __syncthreads();
    uint64_t* sums = vw.sum + (size_t)r * P.NT;
    if (tid < 64) {
        // the tiles' sums go out by exchanges, which are back when they are where every XCD
        // reads them; then the count.  (A release and acquire at device scope write back and
        // invalidate whole caches: the kernel took 150 us for 133 refusals with them.)
        const int tile = lo / kTile + tid;
        if (tid < TPS && tile < P.NT) {
            uint64_t part = 0;
#pragma unroll
            for (int i = 0; i < WV; ++i) part += tile_part[tid][i];
            uint64_t before = __hip_atomic_exchange(&sums[tile], part, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            asm volatile("" : "+v"(before));
        }
    }
    if (!arrive_last(&vw.arrived[r], (uint32_t)spans, &last)) return;

    // the last span to arrive: the tile the draw lands in, then the token
    {
        static_assert(kMaxTiles <= kVerThreads, "a thread a tile");
        const uint64_t x = tid < P.NT ? from_all(&sums[tid]) : 0ull;
        uint64_t incl = dwave_incl_scan_u64(x);
        if ((tid & 63) == 63) red[tid >> 6] = incl;
        if (tid == 0) found = 0xFFFFFFFFu;
        __syncthreads();
        uint64_t total = 0;
#pragma unroll
        for (int i = 0; i < WV; ++i) {
            if (i < (tid >> 6)) incl += red[i];
            total += red[i];
        }
        uint64_t goal = J.u > 0.0 ? (uint64_t)(J.u * (double)total) : 0;
        if (goal >= total) goal = total - 1;
        if (total && incl - x <= goal && goal < incl) { found = (uint32_t)tid; left = goal - (incl - x); }
    }
    __syncthreads();
    if (found == 0xFFFFFFFFu) {
        // nothing: the most likely token, as FINISH has it, or the first of those that a row
        // settled by its mass alone has at its largest scaled logit
        uint32_t best = 0xFFFFFFFFu;
        if (mass_only(a, row, a.flags[row])) {
            const float M = P.w.res[row].M;
            if (tid == 0 && m0 == M) best = 0;
            for (int l = 0; l < V; l += kSpanV) {
                if (R.pen) R.count(l);
                for (int i = l + tid; i < min(l + kSpanV, V); i += kVerThreads) {
                    float x = load_elem<DT>(R.rowp, (uint32_t)i);
                    if (R.pen && cnt[i - l]) x = penalize(x, R.rep, R.pres, R.freq, cnt[i - l]);
                    if (i > 0 && row_scale(x, J.s) == M && (uint32_t)i < best) best = (uint32_t)i;
                }
            }
            best = block_min_u32<kVerThreads>(best, (uint32_t*)red);
        }
        if (tid == 0) *J.out = best < (uint32_t)V ? (int64_t)best : a.tokens[row];
        return;
    }
    const int at = (int)found * kTile;
    if (R.pen) R.count(at);
    const float m = R.mt[1 + found], share = share_of(R.ct[1 + found], J.total);
    uint4 raw[GPT];
    DraftVec<QT, EPL> qs[GPT];
#pragma unroll
    for (int j = 0; j < GPT; ++j) {
        const int e0 = at + (j * kVerThreads + tid) * EPL;
        raw[j] = R.load(e0);
        if constexpr (QT >= 0) qs[j].load(qp, e0, V);
    }
    uint64_t goal = left;
#pragma unroll
    for (int j = 0; j < GPT; ++j) {
        const int e0 = at + (j * kVerThreads + tid) * EPL;
        Excess w[EPL];
        excess(at, e0, m, share, raw[j], qs[j], true, w);
        uint64_t mine = 0;
#pragma unroll
        for (int e = 0; e < EPL; ++e) mine += ((uint64_t)w[e].hi << 24) + w[e].lo;
        const uint64_t incl = dwave_incl_scan_u64(mine);
        __syncthreads();
        if ((tid & 63) == 63) red[tid >> 6] = incl;
        __syncthreads();
        uint64_t b = incl - mine, sum = 0;
#pragma unroll
        for (int i = 0; i < WV; ++i) {
            if (i < (tid >> 6)) b += red[i];
            sum += red[i];
        }
        if (b <= goal && goal < b + mine) {                    // one thread
#pragma unroll
            for (int e = 0; e < EPL; ++e) {
                const uint64_t x = ((uint64_t)w[e].hi << 24) + w[e].lo;
                if (b <= goal && goal < b + x) *J.out = e0 + e;
                b += x;
            }
        }
        if (goal < sum) return;                                // the same in every thread
        goal -= sum;
    }
}

}  // namespace fie
