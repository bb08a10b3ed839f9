// Verification of drafted tokens behind the sampler's kernels (fie_sampler_verify).
//
// k_accept tests a request's drafts: p(d_j) from the row's thresholds, tile maxima and kept
// mass, which the sampler left in the workspace.  k_refused draws the token of a refusal from
// what the row's p has over the draft's q, over one row of logits and one of q a request:
// 8192-token spans sum the excess as whole numbers (fixed point, 2^-48: sums have no order),
// and the last span of a request to arrive finds the span and the token the draw lands in.
#pragma once

#include "launchers.h"

namespace fie {

constexpr int kVerThreads = 256;
constexpr int kVerSpan = 8192;             // tokens a workgroup of k_refused

// What k_accept leaves for k_refused, in workspace arrays that the sampler is done with.
struct VerWs {
    int32_t* at;        // [requests] the refused draft, -1: nothing left to draw
    uint32_t* arrived;  // [requests]
    uint64_t* sum;      // [requests * spans]
};

// A row's distribution as the sampler left it.
struct RowDist {
    RowRes rr;
    double total;
    const float* mt;
    const uint64_t* ct;
    float edge;         // tokens above it are kept, those at it up to token `lim`
    int lim;

    FIE_DEV RowDist(const KParams& P, int row)
        : rr(P.w.res[row]), mt(P.w.mt + (size_t)row * (P.NT + 1)), ct(P.w.ct + (size_t)row * (P.NT + 1))
    {
        total = u128_to_double(((u128)rr.khi << 64) | rr.klo);
        // kept is: key >= tau and (key, index) >= cut in rank order; the later of the two decides
        const uint32_t ck = comp_k(rr.cut);
        const bool at_cut = rr.cut != 0 && ck >= rr.tau;
        const uint32_t k = at_cut ? ck : rr.tau;
        edge = k > kKeyNegInf ? key_to_float(k) : -__builtin_inff();
        lim = at_cut ? (int)comp_idx(rr.cut) : 0x7FFFFFFF;
    }
    // a slot's share of the kept mass per unit of weight
    FIE_DEV float share(int slot) const { return total > 0.0 ? (float)((double)ct[slot] / total) : 0.0f; }
    FIE_DEV bool kept(float y, int idx) const { return y > edge || (y == edge && idx <= lim); }
    // weight20(d) 2^20 floored is the token's weight, below 2^41
    FIE_DEV float prob(float y, int idx, float m, float sh) const
    {
        return kept(y, idx) ? __builtin_floorf(weight20(y - m) * 0x1p20f) * sh : 0.0f;
    }
};

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

// One workgroup a request: draft j by thread j; on rows with penalties the draft's
// occurrences in the row's history are counted first, a wave a draft.
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
        if (tid == 0) { v.accepted[r] = -1; vw.at[r] = -1; }
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
            const RowDist D(P, row);
            if (D.rr.greedy) {
                p = id == D.rr.token ? 1.0f : 0.0f;
            } else {
                float y = D.mt[0];
                int slot = 0;
                if (id != 0) {
                    float x = load_elem<DT>((const char*)a.logits + (size_t)row * (size_t)a.row_stride * DTy<DT>::SZ, (uint32_t)id);
                    if (a.apply_penalties && cnt[tid]) x = penalize(x, a.repetition[row], a.presence[row], a.frequency[row], cnt[tid]);
                    y = row_scale(x, D.rr.s);
                    slot = 1 + (int)id / kTile;
                }
                p = D.prob(y, (int)id, D.mt[slot], D.share(slot));
            }
            qd = v.draft_probs ? draft_prob(v, q.first + tid, id) : 1.0f;
        }
        if (v.target_probs) v.target_probs[q.first + tid] = p;
        const double u = row_uniform(a, row, fl & ~FIE_FLAG_NO_DRAW);
        if (!(u * (double)qd < (double)p)) refused = (uint32_t)tid;
    }
    const int n = (int)min(block_min_u32<kVerThreads>(refused, red), (uint32_t)q.k);
    if (tid < n) out[tid] = id;
    if (tid > n && tid <= v.max_drafts) out[tid] = -1;
    if (tid == 0) {
        v.accepted[r] = n;
        vw.arrived[r] = 0;
        // no draw left: every draft kept, or a greedy row
        const bool done = n == q.k || P.w.res[q.row + n].greedy;
        vw.at[r] = done ? -1 : n;
        if (done) out[n] = a.tokens[q.row + n];
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
// of them is kept.
template <int DT, int QT>
__global__ __launch_bounds__(kVerThreads) void k_refused(const KParams P, const fie_verify_args v, const VerWs vw)
{
    constexpr int EPL = DTy<DT>::EPL, SZ = DTy<DT>::SZ, NL = kVerSpan / kVerThreads / EPL;
    __shared__ uint32_t cnt[kVerSpan];
    __shared__ uint64_t red[kVerThreads / 64];
    __shared__ uint64_t left;
    __shared__ uint32_t found, last;
    const fie_sampler_args& a = P.a;
    const int r = blockIdx.y, tid = threadIdx.x, V = a.vocab, spans = gridDim.x;
    const int n = vw.at[r];
    if (n < 0) return;
    Request q;
    request_of(P, v, r, &q);
    const int row = q.row + n;
    const RowDist D(P, row);
    const bool pen = a.apply_penalties && (a.flags[row] & FIE_FLAG_PENALTY);
    const float rep = pen ? a.repetition[row] : 1.0f, pres = pen ? a.presence[row] : 0.0f, freq = pen ? a.frequency[row] : 0.0f;
    const int64_t draft = v.draft_ids[q.first + n];
    const char* rowp = (const char*)a.logits + (size_t)row * (size_t)a.row_stride * SZ;
    const char* qp = nullptr;
    if constexpr (QT >= 0) qp = (const char*)v.draft_probs + (size_t)(q.first + n) * (size_t)v.draft_stride * DTy<QT>::SZ;
    // the divide by Markstein's correction where it is exact, and where neither answer counts
    // (an infinite logit's weight is 0 either way)
    const float s = D.rr.s, rs = 1.0f / s;
    const bool quick = s >= 0x1p-30f && s <= 0x1p30f;
    const bool all = D.edge == -__builtin_inff() && D.lim == 0x7FFFFFFF;     // no filter

    auto count = [&](int lo) {             // the span's penalty counts
        __syncthreads();
        for (int i = tid; i < kVerSpan; i += kVerThreads) cnt[i] = 0;
        __syncthreads();
        const int64_t h1 = hist_end(a, row);
        for (int64_t h = a.hist_offsets[row] + tid; h < h1; h += kVerThreads) {
            const uint32_t id = (uint32_t)a.hist_ids[h];
            if (id >= (uint32_t)lo && id - (uint32_t)lo < (uint32_t)kVerSpan && id < (uint32_t)V) atomicAdd(&cnt[id - lo], 1u);
        }
        __syncthreads();
    };
    // the tile of the EPL tokens from e0 on holds none that is kept (one tile a workgroup)
    auto below = [&](int e0) { return e0 >= V || D.mt[1 + e0 / kTile] < D.edge; };
    // what p has over q at them, from the logits as loaded
    auto excess = [&](int lo, int e0, uint4 raw, DraftVec<QT, EPL> dv, bool have_q, Excess (&w)[EPL]) {
        const int slot = 1 + min(e0, V - 1) / kTile;
        const float m = D.mt[slot], sh = D.share(slot);
        float y[EPL];
        bool odd = false, any = false;
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
            float x = lane_get<DT>(raw, e);
            if (pen && e0 + e < V && cnt[e0 + e - lo]) x = penalize(x, rep, pres, freq, cnt[e0 + e - lo]);
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
        if (e0 == 0) y[0] = D.mt[0];
#pragma unroll
        for (int e = 0; e < EPL; ++e) any |= D.kept(y[e], e0 + e);
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
            float p = D.prob(y[e], idx, m, sh);
            if (idx == 0) p = D.prob(y[0], 0, y[0], D.share(0));
            float qv;
            if constexpr (QT >= 0) qv = dv.get(e);
            else qv = idx == draft ? 1.0f : 0.0f;
            w[e] = excess_of(idx < V ? p : 0.0f, qv);
        }
    };

    const int lo = blockIdx.x * kVerSpan;
    if (pen) count(lo);
    uint32_t hi = 0, lw = 0;
    uint4 raw[NL];
    DraftVec<QT, EPL> qs[NL];
#pragma unroll
    for (int j = 0; j < NL; ++j) {
        const int g0 = lo + j * kVerThreads * EPL;
        raw[j] = make_uint4(0, 0, 0, 0);
        if (!below(g0) || g0 == 0) {                // token 0 is a tile of its own
            raw[j] = load_group<DT>(rowp, g0 + tid * EPL, V);
            if constexpr (QT >= 0)
                if (all) qs[j].load(qp, g0 + tid * EPL, V);
        }
    }
#pragma unroll
    for (int j = 0; j < NL; ++j) {
        const int g0 = lo + j * kVerThreads * EPL;
        if (below(g0) && g0 != 0) continue;
        Excess w[EPL];
        excess(lo, g0 + tid * EPL, raw[j], qs[j], all, w);
#pragma unroll
        for (int e = 0; e < EPL; ++e) { hi += w[e].hi; lw += w[e].lo; }
    }
    const uint64_t part = block_sum_u64<kVerThreads>(((uint64_t)hi << 24) + lw, red);
    uint64_t* sums = vw.sum + (size_t)r * spans;
    if (tid == 0) {
        // the sum goes out by an exchange, which is back when it is where every XCD reads it;
        // then the count.  (A release and acquire at device scope write back and invalidate
        // whole caches: the kernel took 150 us for 133 refusals with them.)
        uint64_t before = __hip_atomic_exchange(&sums[blockIdx.x], part, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("s_waitcnt vmcnt(0)" : "+v"(before)::"memory");
        last = __hip_atomic_fetch_add(&vw.arrived[r], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)spans - 1;
    }
    __syncthreads();
    if (!last) return;

    // the last span to arrive: the span the draw lands in, then the token (at most 64 spans)
    if (tid < 64) {
        const uint64_t x = tid < spans ? __hip_atomic_load(&sums[tid], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0ull;
        const uint64_t incl = dwave_incl_scan_u64(x);
        const uint64_t total = shfl_u64(incl, 63);
        if (total) {
            const int32_t fl = a.flags[q.row + q.k] & ~FIE_FLAG_NO_DRAW;
            const double u = row_uniform(a, q.row + q.k, fl);
            uint64_t goal = u > 0.0 ? (uint64_t)(u * (double)total) : 0;
            if (goal >= total) goal = total - 1;
            const uint64_t over = __ballot(incl > goal);
            if (tid == (int)__builtin_ctzll(over)) { found = (uint32_t)tid; left = goal - (incl - x); }
        } else if (tid == 0) {
            found = 0xFFFFFFFFu;
        }
    }
    __syncthreads();
    int64_t* out = v.tokens + (size_t)r * (v.max_drafts + 1) + n;
    if (found == 0xFFFFFFFFu) {
        // nothing: the most likely token, as FINISH has it, or the first of those that a row
        // settled by its mass alone has at its largest scaled logit
        uint32_t best = 0xFFFFFFFFu;
        if (mass_only(a, row, a.flags[row])) {
            if (tid == 0 && D.mt[0] == D.rr.M) best = 0;
            for (int l = 0; l < V; l += kVerSpan) {
                if (pen) count(l);
                for (int i = l + tid; i < min(l + kVerSpan, V); i += kVerThreads) {
                    float x = load_elem<DT>(rowp, (uint32_t)i);
                    if (pen && cnt[i - l]) x = penalize(x, rep, pres, freq, cnt[i - l]);
                    if (i > 0 && row_scale(x, s) == D.rr.M && (uint32_t)i < best) best = (uint32_t)i;
                }
            }
            best = block_min_u32<kVerThreads>(best, (uint32_t*)red);
        }
        if (tid == 0) *out = best < (uint32_t)V ? (int64_t)best : a.tokens[row];
        return;
    }
    const int at = (int)found * kVerSpan;
    if (pen) count(at);
    uint64_t goal = left;
#pragma unroll
    for (int j = 0; j < NL; ++j) raw[j] = load_group<DT>(rowp, at + (j * kVerThreads + tid) * EPL, V);
#pragma unroll
    for (int j = 0; j < NL; ++j) {
        const int e0 = at + (j * kVerThreads + tid) * EPL;
        Excess w[EPL];
        excess(at, e0, raw[j], qs[j], false, w);
        uint64_t mine = 0;
#pragma unroll
        for (int e = 0; e < EPL; ++e) mine += ((uint64_t)w[e].hi << 24) + w[e].lo;
        const uint64_t incl = dwave_incl_scan_u64(mine);
        __syncthreads();
        if ((tid & 63) == 63) red[tid >> 6] = incl;
        __syncthreads();
        uint64_t before = 0, sum = 0;
        for (int i = 0; i < kVerThreads / 64; ++i) {
            if (i < (tid >> 6)) before += red[i];
            sum += red[i];
        }
        before += incl - mine;
        if (before <= goal && goal < before + mine) {          // one thread of one round
            uint64_t b = before;
#pragma unroll
            for (int e = 0; e < EPL; ++e) {
                const uint64_t x = ((uint64_t)w[e].hi << 24) + w[e].lo;
                if (b <= goal && goal < b + x) *out = e0 + e;
                b += x;
            }
        }
        if (goal < sum) return;                                // the same in every thread
        goal -= sum;
    }
}

}  // namespace fie
