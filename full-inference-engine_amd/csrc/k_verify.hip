// Instantiations of the verification's kernels (verify.h) and their launcher.
#include "verify.h"

namespace fie {

template <int DT>
static void verify_dt(const KParams& P, const fie_verify_args& v, const VerWs& vw, hipStream_t st)
{
    k_accept<DT><<<v.requests, kVerThreads, 0, st>>>(P, v, vw);
    if (P.a.rows == v.requests && !v.draws) return;         // no drafts, no refusals
    const dim3 grid((P.a.vocab + kVerSpan - 1) / kVerSpan, v.requests);
    const size_t lds = P.a.apply_penalties ? kVerSpan * sizeof(uint32_t) : 0;
    if (!v.draft_probs) k_refused<DT, -1><<<grid, kVerThreads, lds, st>>>(P, v, vw);
    else if (v.draft_dtype == FIE_F32) k_refused<DT, FIE_F32><<<grid, kVerThreads, lds, st>>>(P, v, vw);
    else if (v.draft_dtype == FIE_F16) k_refused<DT, FIE_F16><<<grid, kVerThreads, lds, st>>>(P, v, vw);
    else k_refused<DT, FIE_BF16><<<grid, kVerThreads, lds, st>>>(P, v, vw);
    if (!v.draws) return;
    k_rank<DT, 2><<<grid, kVerThreads, lds, st>>>(P, vw);
    k_rank<DT, 3><<<grid, kVerThreads, lds, st>>>(P, vw);
}

hipError_t launch_verify(const KParams& P, const fie_verify_args& v, hipStream_t st)
{
    // the candidates' and deferred rows' arrays are free once the rows are settled: a request has at least one
    // row, and a row at least as many tiles as spans
    const VerWs vw{(VerJob*)P.w.dfr, P.w.ncand, P.w.sw, P.w.maxc};
    switch (P.a.dtype) {
    case FIE_F32: verify_dt<FIE_F32>(P, v, vw, st); break;
    case FIE_F16: verify_dt<FIE_F16>(P, v, vw, st); break;
    default: verify_dt<FIE_BF16>(P, v, vw, st); break;
    }
    return hipGetLastError();
}

}  // namespace fie
