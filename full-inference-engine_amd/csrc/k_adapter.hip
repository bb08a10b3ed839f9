// Low-rank adapters behind the C ABI of include/fie_decode.h.
#include <algorithm>

#include "adapter.h"

namespace fie {

static int64_t plan_most(int64_t tokens, int64_t adapters) { return tokens / kTileTokens + std::min(tokens, adapters + 1); }

constexpr int kDownSteps = 4;                           // of a wave at a time; 2 of 64 ranks (4001 x 4096 22 us, 24 with 4)

static AdapterWork adapter_work(const fie_adapter_args& a)
{
    AdapterWork w;
    w.h = (float*)a.workspace;
    w.most = (int)plan_most(a.tokens, a.adapters);
    // enough workgroups to fill the CUs, as long as each wave has its steps of k
    const int step = (a.dtype == FIE_F32 ? 16 : 32) * kDownSteps * kDownWaves;
    w.splits = std::max(1, std::min({(a.k + step - 1) / step, 1024 / std::max(w.most, 1), 16}));
    return w;
}

static size_t adapter_bytes(const fie_adapter_args& a) { return (size_t)adapter_work(a).splits * a.tokens * a.rank * 4; }

template <int DX, int DT, bool ALIGNED>
static hipError_t down_of(const fie_adapter_args& a, const AdapterWork& w, hipStream_t st)
{
    const dim3 grid((unsigned)w.splits, (unsigned)w.most);
    if (a.rank <= 16) k_adapter_down<DX, DT, 1, kDownSteps, ALIGNED><<<grid, 64 * kDownWaves, 0, st>>>(a, w);
    else if (a.rank <= 32) k_adapter_down<DX, DT, 2, kDownSteps, ALIGNED><<<grid, 64 * kDownWaves, 0, st>>>(a, w);
    else if (a.rank <= 48) k_adapter_down<DX, DT, 3, kDownSteps, ALIGNED><<<grid, 64 * kDownWaves, 0, st>>>(a, w);
    else k_adapter_down<DX, DT, 4, 2, ALIGNED><<<grid, 64 * kDownWaves, 0, st>>>(a, w);
    return hipGetLastError();
}

template <int DX, int DT>
static hipError_t down(const fie_adapter_args& a, const AdapterWork& w, hipStream_t st)
{
    constexpr int XS = DX == FIE_I8 ? 1 : Operand<DT>::SIZE, BYTES = XS * Operand<DT>::EACH;
    const bool aligned = (uintptr_t)a.x % BYTES == 0 && a.x_stride * XS % BYTES == 0;
    return aligned ? down_of<DX, DT, true>(a, w, st) : down_of<DX, DT, false>(a, w, st);
}

template <int DT, int DY, int DB>
static hipError_t up(const fie_adapter_args& a, const AdapterWork& w, hipStream_t st)
{
    constexpr int YB = DY == FIE_F32 ? 16 : 8, BB = DB == FIE_F32 ? 16 : 8;
    const int wide = (uintptr_t)a.base % BB == 0 && a.base_stride % 4 == 0 && (uintptr_t)a.y % YB == 0 && a.y_stride % 4 == 0;
    const int blocks = (a.n + kUpChannels - 1) / kUpChannels;
    // as many waves as the CUs hold (16 each), and then more steps each
    const int steps = (int)std::max<int64_t>(1, std::min<int64_t>(8, (int64_t)blocks * w.most / (16 * std::max(cu_count(), 1))));
    const dim3 grid((unsigned)((blocks + steps - 1) / steps), (unsigned)((w.most + kUpWaves - 1) / kUpWaves));
    switch (a.rank / 16) {
    case 1: k_adapter_up<DT, DY, DB, 1><<<grid, 64 * kUpWaves, 0, st>>>(a, w, wide, steps); break;
    case 2: k_adapter_up<DT, DY, DB, 2><<<grid, 64 * kUpWaves, 0, st>>>(a, w, wide, steps); break;
    case 3: k_adapter_up<DT, DY, DB, 3><<<grid, 64 * kUpWaves, 0, st>>>(a, w, wide, steps); break;
    case 4: k_adapter_up<DT, DY, DB, 4><<<grid, 64 * kUpWaves, 0, st>>>(a, w, wide, steps); break;
    default: k_adapter_up<DT, DY, DB, 0><<<grid, 64 * kUpWaves, 0, st>>>(a, w, wide, steps); break;
    }
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

static int plan_check(int64_t tokens, int64_t adapters)
{
    if (tokens < 0 || tokens > 1 << 24) return fail(FIE_E_ARG, "tokens out of range [0, 16777216]");
    if (adapters < 1 || adapters > FIE_MAX_ADAPTERS) return fail(FIE_E_ARG, "adapters out of range [1, 4096]");
    if (plan_most(tokens, adapters) > 65535) return fail(FIE_E_ARG, "more tiles than a launch holds");
    return FIE_OK;
}

static int adapter_check(const fie_adapter_args* a)
{
    if (!a) return fail(FIE_E_ARG, "args is NULL");
    if (const int rc = plan_check(a->tokens, a->adapters); rc != FIE_OK) return rc;
    if (a->dtype < FIE_F32 || a->dtype > FIE_BF16 || (a->x_dtype != a->dtype && a->x_dtype != FIE_I8))
        return fail(FIE_E_ARG, "x is in the adapters' type or int8");
    if ((a->y_dtype != a->dtype && a->y_dtype != FIE_F32) || (a->base && a->base_dtype != a->y_dtype && a->base_dtype != FIE_F32))
        return fail(FIE_E_ARG, "y is in the adapters' type or fp32, base in y's or fp32");
    if (a->n < 1 || a->n > 0x7FFFFF00 || a->k < 1 || a->k > FIE_MAX_K) return fail(FIE_E_ARG, "n or k out of range");
    if (a->k_pad < a->k || a->k_pad % FIE_ADAPTER_K) return fail(FIE_E_ARG, "k_pad is k's next multiple of 64");
    if (a->rank < FIE_ADAPTER_RANK || a->rank > FIE_MAX_RANK || a->rank % FIE_ADAPTER_RANK)
        return fail(FIE_E_ARG, "rank is a multiple of 16 in [16, 256]");
    if (a->b_pitch < a->rank || a->b_pitch % (a->dtype == FIE_F32 ? 4 : 8)) return fail(FIE_E_ARG, "b_pitch is rank or more, a multiple of 16 bytes");
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

extern "C" size_t fie_adapter_plan_ints(int32_t tokens, int32_t adapters)
{
    if (plan_check(tokens, adapters) != FIE_OK) return 0;
    return kPlanHead + (size_t)plan_most(tokens, adapters) * kPlanTile + tokens;
}

extern "C" int fie_adapter_plan(const fie_adapter_plan_args* a, void* stream)
{
    if (!a) return fail(FIE_E_ARG, "args is NULL");
    if (const int rc = plan_check(a->tokens, a->adapters); rc != FIE_OK) return rc;
    if (!a->plan || (a->tokens && !a->ids)) return fail(FIE_E_ARG, "ids or plan is NULL");
    k_adapter_plan<<<1, kPlanThreads, 0, (hipStream_t)stream>>>(*a, (int)plan_most(a->tokens, a->adapters));
    return launch_status(hipGetLastError(), "k_adapter_plan");
}

extern "C" size_t fie_adapter_workspace_size(const fie_adapter_args* a)
{
    return a && a->tokens > 0 && a->k > 0 && a->rank > 0 && a->adapters > 0 ? adapter_bytes(*a) : 0;
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
