// Instantiations of the verification's kernels (verify.h) and their launcher.
#include "verify.h"

namespace fie {

template <int DT, int TPS>
static void spans_of(const KParams& P, const fie_verify_args& v, const VerWs& vw, hipStream_t st)
{
    constexpr int span = TPS * kTile;
    const dim3 grid((P.a.vocab + span - 1) / span, v.requests);
    const size_t lds = P.a.apply_penalties ? span * sizeof(uint32_t) : 0;
    if (!v.draft_probs) k_refused<DT, -1, TPS><<<grid, kVerThreads, lds, st>>>(P, v, vw);
    else if (v.draft_dtype == FIE_F32) k_refused<DT, FIE_F32, TPS><<<grid, kVerThreads, lds, st>>>(P, v, vw);
    else if (v.draft_dtype == FIE_F16) k_refused<DT, FIE_F16, TPS><<<grid, kVerThreads, lds, st>>>(P, v, vw);
    else k_refused<DT, FIE_BF16, TPS><<<grid, kVerThreads, lds, st>>>(P, v, vw);
    if (!v.draws) return;
    k_rank<DT, 2, TPS><<<grid, kVerThreads, lds, st>>>(P, vw);
    k_rank<DT, 3, TPS><<<grid, kVerThreads, lds, st>>>(P, vw);
}

template <int DT>
static void verify_dt(const KParams& P, const fie_verify_args& v, const VerWs& vw, hipStream_t st)
{
    k_accept<DT><<<v.requests, kVerThreads, 0, st>>>(P, v, vw);
    if (P.a.rows == v.requests && !v.draws) return;         // no drafts, no refusals
    // A wave takes a 2048-token tile's part in 1 us and four tiles' in 4: with few requests a
    // tile a workgroup is a shorter way, with many the workgroups' own steps (6 us) count.  us a
    // call, a tile and four tiles a workgroup, at vocab 151936: 1 request 40, 42.5; 16 81, 88; 32
    // 97, 102; 64 142, 137; 256 327, 301.
    if ((int64_t)P.NS * v.requests <= 4 * cu_count()) spans_of<DT, 1>(P, v, vw, st);
    else spans_of<DT, kVerTiles>(P, v, vw, st);
}

hipError_t launch_verify(const KParams& P, const fie_verify_args& v, hipStream_t st)
{
    // the candidates' and deferred rows' arrays are free once the rows are settled: a request has at least one
    // row, and a row at least as many tiles as spans
    const VerWs vw{(VerJob*)P.w.dfr, P.w.ncand, P.w.sw};
    switch (P.a.dtype) {
    case FIE_F32: verify_dt<FIE_F32>(P, v, vw, st); break;
    case FIE_F16: verify_dt<FIE_F16>(P, v, vw, st); break;
    default: verify_dt<FIE_BF16>(P, v, vw, st); break;
    }
    return hipGetLastError();
}

}  // namespace fie
