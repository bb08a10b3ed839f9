// Low-rank adapters behind the C ABI of include/fie_decode.h.
#include <algorithm>

#include "adapter.h"

namespace fie {

static int plan_most(int64_t tokens, int64_t adapters, int tile) { return (int)(tokens / tile + std::min(tokens, adapters + 1)); }

static AdapterWork adapter_work(const fie_adapter_args& a)
{
    AdapterWork w;
    w.h = (float*)a.workspace;
    w.most = plan_most(a.tokens, a.adapters, a.tile);
    // enough workgroups to fill the CUs; each wave has its steps of k
    const int step = (a.dtype == FIE_F32 ? 16 : 32) * kDownSteps * kDownWaves;
    w.splits = std::max(1, std::min({(a.k + step - 1) / step, 512 / std::max(w.most, 1), 32}));
    return w;
}

static size_t adapter_bytes(const fie_adapter_args& a)
{
    return (size_t)adapter_work(a).splits * a.tokens * a.rank * 4;
}

template <int DX, int DT, int MT, bool ALIGNED>
static hipError_t down_of(const fie_adapter_args& a, const AdapterWork& w, hipStream_t st)
{
    const dim3 grid((unsigned)w.splits, (unsigned)w.most);
    if (a.rank <= 16) k_adapter_down<DX, DT, MT, 1, ALIGNED><<<grid, 64 * kDownWaves, 0, st>>>(a, w);
    else if (a.rank <= 32) k_adapter_down<DX, DT, MT, 2, ALIGNED><<<grid, 64 * kDownWaves, 0, st>>>(a, w);
    else k_adapter_down<DX, DT, MT, 4, ALIGNED><<<grid, 64 * kDownWaves, 0, st>>>(a, w);
    return hipGetLastError();
}

template <int DX, int DT>
static hipError_t down(const fie_adapter_args& a, const AdapterWork& w, hipStream_t st)
{
    constexpr int XS = DX == FIE_I8 ? 1 : Operand<DT>::SIZE, BYTES = XS * Operand<DT>::EACH;
    const bool aligned = (uintptr_t)a.x % BYTES == 0 && a.x_stride * XS % BYTES == 0;
    if (a.tile == 16) return aligned ? down_of<DX, DT, 1, true>(a, w, st) : down_of<DX, DT, 1, false>(a, w, st);
    return aligned ? down_of<DX, DT, 4, true>(a, w, st) : down_of<DX, DT, 4, false>(a, w, st);
}

template <int DT, int DY, int DB>
static hipError_t up(const fie_adapter_args& a, const AdapterWork& w, hipStream_t st)
{
    constexpr int YB = DY == FIE_F32 ? 16 : 8, BB = DB == FIE_F32 ? 16 : 8;
    const int wide = ((uintptr_t)a.base % BB == 0 && a.base_stride % 4 == 0 ? 1 : 0) | ((uintptr_t)a.y % YB == 0 && a.y_stride % 4 == 0 ? 2 : 0);
    const dim3 grid((unsigned)((a.n + kUpChannels - 1) / kUpChannels), (unsigned)w.most);
    const size_t lds = (size_t)a.tile * (a.rank + 4) * 4;
    if (a.tile == 16) k_adapter_up<DT, DY, DB, 1><<<grid, 64 * kUpWaves, lds, st>>>(a, w, wide);
    else k_adapter_up<DT, DY, DB, 4><<<grid, 64 * kUpWaves, lds, st>>>(a, w, wide);
    return hipGetLastError();
}

template <int DT>
static hipError_t adapter_dt(const fie_adapter_args& a, hipStream_t st)
{
    const AdapterWork w = adapter_work(a);
    hipError_t e = a.x_dtype == FIE_I8 ? down<FIE_I8, DT>(a, w, st) : down<DT, DT>(a, w, st);
    if (e != hipSuccess) return e;
    if (a.y_dtype == FIE_F32) return up<DT, FIE_F32, FIE_F32>(a, w, st);
    if constexpr (DT != FIE_F32) return a.base_dtype == FIE_F32 ? up<DT, DT, FIE_F32>(a, w, st) : up<DT, DT, DT>(a, w, st);
    return hipSuccess;
}

static int plan_check(int64_t tokens, int64_t adapters, int tile)
{
    if (tokens < 0 || tokens > 1 << 24) return fail(FIE_E_ARG, "tokens out of range [0, 16777216]");
    if (adapters < 1 || adapters > FIE_MAX_ADAPTERS) return fail(FIE_E_ARG, "adapters out of range [1, 4096]");
    if (tile != 16 && tile != 64) return fail(FIE_E_ARG, "tile is 16 or 64");
    if (plan_most(tokens, adapters, tile) > 65535) return fail(FIE_E_ARG, "more tiles than a launch holds");
    return FIE_OK;
}

static int adapter_check(const fie_adapter_args* a)
{
    if (!a) return fail(FIE_E_ARG, "args is NULL");
    if (const int rc = plan_check(a->tokens, a->adapters, a->tile); rc != FIE_OK) return rc;
    if (a->dtype < FIE_F32 || a->dtype > FIE_BF16 || (a->x_dtype != a->dtype && a->x_dtype != FIE_I8))
        return fail(FIE_E_ARG, "x is in the adapters' type or int8");
    if ((a->y_dtype != a->dtype && a->y_dtype != FIE_F32) || (a->base && a->base_dtype != a->y_dtype && a->base_dtype != FIE_F32))
        return fail(FIE_E_ARG, "y is in the adapters' type or fp32, base in y's or fp32");
    if (a->n < 1 || a->n > 0x7FFFFF00 || a->k < 1 || a->k > FIE_MAX_K) return fail(FIE_E_ARG, "n or k out of range");
    if (a->k_pad < a->k || a->k_pad % FIE_ADAPTER_K) return fail(FIE_E_ARG, "k_pad is k's next multiple of 64");
    if (a->rank < FIE_ADAPTER_RANK || a->rank > FIE_MAX_RANK || a->rank % FIE_ADAPTER_RANK)
        return fail(FIE_E_ARG, "rank is a multiple of 16 in [16, 256]");
    if (a->x_stride < 0 || a->y_stride < a->n) return fail(FIE_E_ARG, "a row stride is shorter than its row");
    if (a->tokens == 0) return FIE_OK;
    if (!a->x || !a->a || !a->b || !a->scale || !a->ranks || !a->plan || !a->y || (a->x_dtype == FIE_I8) != (a->x_scale != nullptr))
        return fail(FIE_E_ARG, "a required pointer is NULL, or x_scale without int8");
    if ((((uintptr_t)a->a | (uintptr_t)a->b) & 15) != 0) return fail(FIE_E_ARG, "adapters not 16-byte aligned");
    if (a->base == a->y && (a->base_dtype != a->y_dtype || a->base_stride != a->y_stride)) return fail(FIE_E_ARG, "base in y's place is in y's type");
    if (!a->workspace || a->workspace_bytes < adapter_bytes(*a)) return fail(FIE_E_WORKSPACE, "workspace too small");
    if (((uintptr_t)a->workspace & 15) != 0) return fail(FIE_E_WORKSPACE, "workspace not 16-byte aligned");
    return FIE_OK;
}

}  // namespace fie

using namespace fie;

extern "C" size_t fie_adapter_plan_ints(int32_t tokens, int32_t adapters, int32_t tile)
{
    if (plan_check(tokens, adapters, tile) != FIE_OK) return 0;
    return kPlanHead + (size_t)plan_most(tokens, adapters, tile) * kPlanTile + tokens;
}

extern "C" int fie_adapter_plan(const fie_adapter_plan_args* a, void* stream)
{
    if (!a) return fail(FIE_E_ARG, "args is NULL");
    if (const int rc = plan_check(a->tokens, a->adapters, a->tile); rc != FIE_OK) return rc;
    if (!a->plan || (a->tokens && !a->ids)) return fail(FIE_E_ARG, "ids or plan is NULL");
    k_adapter_plan<<<1, kPlanThreads, 0, (hipStream_t)stream>>>(*a, plan_most(a->tokens, a->adapters, a->tile));
    return launch_status(hipGetLastError(), "k_adapter_plan");
}

extern "C" size_t fie_adapter_workspace_size(const fie_adapter_args* a)
{
    return a && a->tokens > 0 && a->k > 0 && a->rank > 0 && (a->tile == 16 || a->tile == 64) ? adapter_bytes(*a) : 0;
}

extern "C" int fie_adapter_linear(const fie_adapter_args* a, void* stream)
{
    const int rc = adapter_check(a);
    if (rc != FIE_OK || a->tokens == 0) return rc;
    const hipStream_t st = (hipStream_t)stream;
    switch (a->dtype) {
    case FIE_F32: return launch_status(adapter_dt<FIE_F32>(*a, st), "k_adapter");
    case FIE_F16: return launch_status(adapter_dt<FIE_F16>(*a, st), "k_adapter");
    default: return launch_status(adapter_dt<FIE_BF16>(*a, st), "k_adapter");
    }
}
