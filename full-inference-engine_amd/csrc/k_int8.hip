// The 8-bit integer product behind the C ABI of include/fie_ops.h: instantiations of int8.h's
// kernels and the choice among them.
#include "int8.h"

namespace fie {

template <int DT, int WM, int WN>
static hipError_t tile_of(const fie_int8_args& a, int wide, hipStream_t st)
{
    constexpr int BM = 64 * WM, BN = 64 * WN;
    const int64_t nrb = (a.m + BM - 1) / BM, tiles = (a.n + BN - 1) / BN;
    k_int8_tile<DT, WM, WN><<<(unsigned)(8 * ((tiles + 7) / 8) * nrb), 64 * WM * WN, 0, st>>>(a, (int)nrb, wide);
    return hipGetLastError();
}

template <int DT>
static hipError_t int8_dt(const fie_int8_args& a, hipStream_t st)
{
    constexpr int SZ = DT == FIE_F32 ? 4 : 2;
    const int wide = ((uintptr_t)a.y % (4 * SZ)) == 0 && a.y_stride % 4 == 0;
    if (a.m <= 64) return tile_of<DT, 1, 4>(a, wide, st);
    return tile_of<DT, 2, 2>(a, wide, st);
}

static int int8_check(const fie_int8_args* a)
{
    if (!a) return fail(FIE_E_ARG, "args is NULL");
    if (a->m < 0 || a->m > 0x7FFFFF00 || a->n < 1) return fail(FIE_E_ARG, "sizes out of range");
    if (a->k < 1 || a->k > FIE_MAX_K) return fail(FIE_E_ARG, "k out of range [1, 131071]");
    if (a->y_dtype < FIE_F32 || a->y_dtype > FIE_BF16) return fail(FIE_E_ARG, "unknown dtype");
    if (a->x_stride < a->k || a->w_stride < a->k || a->y_stride < a->n) return fail(FIE_E_ARG, "a row stride is shorter than its row");
    if ((a->m + 63) / 64 * ((a->n + 63) / 64) > 0x0FFFFFFF) return fail(FIE_E_ARG, "m x n too large for one launch");
    if (a->m == 0) return FIE_OK;
    if (!a->x || !a->w || !a->x_scale || !a->w_scale || !a->y) return fail(FIE_E_ARG, "a required pointer is NULL");
    return FIE_OK;
}

}  // namespace fie

using namespace fie;

extern "C" int fie_int8_linear(const fie_int8_args* a, void* stream)
{
    const int rc = int8_check(a);
    if (rc != FIE_OK || a->m == 0) return rc;
    hipStream_t st = (hipStream_t)stream;
    hipError_t e;
    switch (a->y_dtype) {
    case FIE_F32: e = int8_dt<FIE_F32>(*a, st); break;
    case FIE_F16: e = int8_dt<FIE_F16>(*a, st); break;
    default: e = int8_dt<FIE_BF16>(*a, st); break;
    }
    return launch_status(e, "k_int8");
}
