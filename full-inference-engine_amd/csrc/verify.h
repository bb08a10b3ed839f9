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

    FIE_DEV RowDist(const KParams& P, int row)
        : rr(P.w.res[row]), mt(P.w.mt + (size_t)row * (P.NT + 1)), ct(P.w.ct + (size_t)row * (P.NT + 1))
    {
        total = u128_to_double(((u128)rr.khi << 64) | rr.klo);
    }
    // a slot's share of the kept mass per unit of weight
    FIE_DEV float share(int slot) const { return total > 0.0 ? (float)((double)ct[slot] / total) : 0.0f; }
    FIE_DEV bool kept(float y, int idx) const
    {
        const uint64_t c = comp_key(fkey(y), (uint32_t)idx);
        return comp_k(c) >= rr.tau && c >= rr.cut;
    }
    FIE_DEV float prob(float y, int idx, float m, float sh) const { return kept(y, idx) ? weight40(y - m) * sh : 0.0f; }
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
        // no draw left: every draft kept, a greedy row, or a row without mass
        const RowRes& rr = P.w.res[q.row + n];
        const bool done = n == q.k || rr.greedy || (rr.klo | rr.khi) == 0;
        vw.at[r] = done ? -1 : n;
        if (done) out[n] = a.tokens[q.row + n];
    }
}

// N tokens of a row of draft probabilities from e0 on; past V: 0.
template <int QT, int N>
FIE_DEV void load_q(float (&q)[N], const char* rowp, int e0, int V)
{
    constexpr int EPL = DTy<QT>::EPL;
    if constexpr (N >= EPL) {
#pragma unroll
        for (int g = 0; g < N / EPL; ++g) {
            const uint4 w = load_group<QT>(rowp, e0 + g * EPL, V);
#pragma unroll
            for (int e = 0; e < EPL; ++e) q[g * EPL + e] = at_least_0(lane_get<QT>(w, e));
        }
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) q[e] = e0 + e < V ? at_least_0(load_elem<QT>(rowp, (uint32_t)(e0 + e))) : 0.0f;
    }
}

// Grid (spans, requests).  QT: the draft's type, -1 without probabilities.
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
    // the excess of p over q at the EPL tokens from e0 on
    auto excess = [&](int lo, int e0, uint64_t (&w)[EPL]) {
        const uint4 raw = load_group<DT>(rowp, e0, V);
        float qs[EPL];
        if constexpr (QT >= 0) load_q<QT, EPL>(qs, qp, e0, V);
        const int slot = 1 + min(e0, V - 1) / kTile;
        const float m = D.mt[slot], sh = D.share(slot);
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
            const int idx = e0 + e;
            float x = lane_get<DT>(raw, e);
            if (pen && idx < V && cnt[idx - lo]) x = penalize(x, rep, pres, freq, cnt[idx - lo]);
            float p = D.prob(row_scale(x, D.rr.s), idx, m, sh);
            if (idx == 0) p = D.prob(D.mt[0], 0, D.mt[0], D.share(0));
            float qv;
            if constexpr (QT >= 0) qv = qs[e];
            else qv = idx == draft ? 1.0f : 0.0f;
            const float d = p - qv;
            w[e] = idx < V && d > 0.0f ? (uint64_t)((double)d * 0x1p48) : 0ull;
        }
    };

    const int lo = blockIdx.x * kVerSpan;
    if (pen) count(lo);
    uint64_t part = 0;
#pragma unroll 1
    for (int j = 0; j < NL; ++j) {
        uint64_t w[EPL];
        excess(lo, lo + (j * kVerThreads + tid) * EPL, w);
#pragma unroll
        for (int e = 0; e < EPL; ++e) part += w[e];
    }
    part = block_sum_u64<kVerThreads>(part, red);
    uint64_t* sums = vw.sum + (size_t)r * spans;
    if (tid == 0) {
        __hip_atomic_store(&sums[blockIdx.x], part, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = __hip_atomic_fetch_add(&vw.arrived[r], 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)spans - 1;
    }
    __syncthreads();
    if (!last) return;

    // the last span to arrive: the span the draw lands in, then the token
    if (tid == 0) {
        uint64_t total = 0;
        for (int s = 0; s < spans; ++s) total += __hip_atomic_load(&sums[s], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        found = 0xFFFFFFFFu;
        if (total) {
            const int32_t fl = a.flags[q.row + q.k] & ~FIE_FLAG_NO_DRAW;
            const double u = row_uniform(a, q.row + q.k, fl);
            uint64_t goal = u > 0.0 ? (uint64_t)(u * (double)total) : 0;
            if (goal >= total) goal = total - 1;
            int s = 0;
            for (; s < spans - 1; ++s) {
                const uint64_t x = __hip_atomic_load(&sums[s], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                if (x > goal) break;
                goal -= x;
            }
            found = (uint32_t)s;
            left = goal;
        }
    }
    __syncthreads();
    int64_t* out = v.tokens + (size_t)r * (v.max_drafts + 1) + n;
    if (found == 0xFFFFFFFFu) {
        if (tid == 0) *out = a.tokens[row];
        return;
    }
    const int at = (int)found * kVerSpan;
    if (pen) count(at);
    uint64_t goal = left;
    for (int j = 0; j < NL; ++j) {
        uint64_t w[EPL], mine = 0;
        const int e0 = at + (j * kVerThreads + tid) * EPL;
        excess(at, e0, w);
#pragma unroll
        for (int e = 0; e < EPL; ++e) mine += w[e];
        const uint64_t incl = dwave_incl_scan_u64(mine);
        __syncthreads();
        if ((tid & 63) == 63) red[tid >> 6] = incl;
        __syncthreads();
        uint64_t before = 0, all = 0;
        for (int i = 0; i < kVerThreads / 64; ++i) {
            if (i < (tid >> 6)) before += red[i];
            all += red[i];
        }
        before += incl - mine;
        if (before <= goal && goal < before + mine) {          // one thread of one round
            uint64_t b = before;
#pragma unroll
            for (int e = 0; e < EPL; ++e) {
                if (b <= goal && goal < b + w[e]) *out = e0 + e;
                b += w[e];
            }
        }
        if (goal < all) return;                                // the same in every thread
        goal -= all;
    }
}

}  // namespace fie
