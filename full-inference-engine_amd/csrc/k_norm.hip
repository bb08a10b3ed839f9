// Block norms behind the C ABI of include/fie_ops.h: instantiations of norm.h's kernel and
// the choice among them.
#include "norm.h"

namespace fie {

template <int DX, int DR, int VPT, bool ONE>
static hipError_t norm_at(const fie_norm_args& a, unsigned grid, int threads, hipStream_t st)
{
    // every load at once where the registers hold them and no parameter needs another type
    // (333 x 2050, layer norms on both sides and a gate: 9.4 us without, 8.5)
    if (VPT <= 2 && (DX == FIE_F32 || !(a.weight_f32 || a.gate_f32)))
        k_norm<DX, DR, VPT, ONE, VPT <= 2><<<grid, threads, 0, st>>>(a);
    else
        k_norm<DX, DR, VPT, ONE, false><<<grid, threads, 0, st>>>(a);
    return hipGetLastError();
}

template <int DX, int DR>
static hipError_t norm_of(const fie_norm_args& a, hipStream_t st)
{
    const int vecs = (a.width + 7) / 8;
    if (a.width > FIE_MAX_WIDTH) {                      // to int8 alone (norm_check)
        k_quantise_wide<DR><<<(unsigned)a.tokens, 1024, 0, st>>>(a);
        return hipGetLastError();
    }
    if (vecs <= 64) return norm_at<DX, DR, 1, true>(a, (unsigned)((a.tokens + 3) / 4), 256, st);
    // Few rows: a vector a thread, the shorter chain (1 x 4096 4.2 us with two, 3.0; 512 x 4096
    // layer 8.2, 7.9); many: two, more in flight a workgroup (1024 x 4096 7.6 with two, 8.4;
    // 8192 x 4096 layer 51, 62).
    const bool few = a.tokens <= 2 * cu_count();
    const int vpt = vecs <= (few ? 512 : 256) ? 1 : vecs <= 1024 ? 2 : vecs <= 4096 ? 4 : 8;
    const int threads = ((vecs + vpt - 1) / vpt + 63) / 64 * 64;
    const unsigned grid = (unsigned)a.tokens;
    switch (vpt) {
    case 1: return norm_at<DX, DR, 1, false>(a, grid, threads, st);
    case 2: return norm_at<DX, DR, 2, false>(a, grid, threads, st);
    case 4: return norm_at<DX, DR, 4, false>(a, grid, threads, st);
    default: return norm_at<DX, DR, 8, false>(a, grid, threads, st);
    }
}

// The rows of one launch: a grid holds fewer than 2^32 threads (past that the launch leaves rows
// out, without an error), and a row takes 64 of them or at most 1024.
static int64_t rows_at_once(int width) { return width <= 512 ? 1 << 25 : 1 << 21; }

static fie_norm_args rows_from(fie_norm_args a, int64_t row)
{
    auto size = [](int dtype) -> int64_t { return dtype == FIE_I8 ? 1 : dtype == FIE_F32 ? 4 : 2; };
    auto on = [&](auto* p, int64_t stride, int64_t bytes) { return p ? (decltype(p))((uintptr_t)p + (uintptr_t)(row * stride * bytes)) : p; };
    a.x = on(a.x, a.x_stride, size(a.x_dtype));
    a.residual = on(a.residual, a.residual_stride, size(a.residual_dtype));
    a.residual_out = on(a.residual_out, a.residual_out_stride, size(a.residual_dtype));
    a.y = on(a.y, a.y_stride, size(a.y_dtype));
    a.y_scale = on(a.y_scale, 1, 4);
    a.gate = on(a.gate, a.gate_stride, a.gate_f32 ? 4 : size(a.x_dtype));
    a.tokens -= row;
    return a;
}

static hipError_t norm_run(const fie_norm_args& a, hipStream_t st)
{
    switch (a.x_dtype * 3 + a.residual_dtype) {
    case FIE_F32 * 3 + FIE_F32: return norm_of<FIE_F32, FIE_F32>(a, st);
    case FIE_F32 * 3 + FIE_F16: return norm_of<FIE_F32, FIE_F16>(a, st);
    case FIE_F32 * 3 + FIE_BF16: return norm_of<FIE_F32, FIE_BF16>(a, st);
    case FIE_F16 * 3 + FIE_F32: return norm_of<FIE_F16, FIE_F32>(a, st);
    case FIE_F16 * 3 + FIE_F16: return norm_of<FIE_F16, FIE_F16>(a, st);
    case FIE_F16 * 3 + FIE_BF16: return norm_of<FIE_F16, FIE_BF16>(a, st);
    case FIE_BF16 * 3 + FIE_F32: return norm_of<FIE_BF16, FIE_F32>(a, st);
    case FIE_BF16 * 3 + FIE_F16: return norm_of<FIE_BF16, FIE_F16>(a, st);
    default: return norm_of<FIE_BF16, FIE_BF16>(a, st);
    }
}

static int norm_check(const fie_norm_args* a)
{
    if (!a) return fail(FIE_E_ARG, "args is NULL");
    if (a->tokens < 0 || a->tokens > 0x7FFFFFFF) return fail(FIE_E_ARG, "tokens out of range");
    const bool alone = !a->x && !a->residual_out && a->kind == FIE_NORM_NONE && a->y && a->y_dtype == FIE_I8;
    if (a->width < 1 || a->width > FIE_MAX_WIDTH)
        if (!alone || a->width < 1 || a->width > FIE_MAX_K)
            return fail(FIE_E_ARG, "width out of range [1, 65536] (a quantisation alone: 131071)");
    if (a->x_dtype < FIE_F32 || a->x_dtype > FIE_BF16 || a->residual_dtype < FIE_F32 || a->residual_dtype > FIE_BF16)
        return fail(FIE_E_ARG, "unknown dtype");
    if (a->x && a->residual_dtype != a->x_dtype && a->residual_dtype != FIE_F32)
        return fail(FIE_E_ARG, "residual is in x's type or fp32");
    if (a->y && a->y_dtype != a->x_dtype && a->y_dtype != FIE_I8) return fail(FIE_E_ARG, "y is in x's type or int8");
    if (a->kind < FIE_NORM_RMS || a->kind > FIE_NORM_NONE) return fail(FIE_E_ARG, "unknown kind of norm");
    if (a->post_norm && (a->kind == FIE_NORM_NONE || !a->x)) return fail(FIE_E_ARG, "post_norm needs x and a kind of norm");
    if (a->gate && (!a->x || (a->gate_step != 0 && a->gate_step != 1))) return fail(FIE_E_ARG, "a gate needs x and a step of 0 or 1");
    if (a->tokens == 0) return FIE_OK;
    if (!a->residual) return fail(FIE_E_ARG, "residual is NULL");
    if (a->y && a->y_dtype == FIE_I8 && !a->y_scale) return fail(FIE_E_ARG, "int8 output without y_scale");
    if (!a->y && !a->residual_out) return fail(FIE_E_ARG, "no output");
    return FIE_OK;
}

}  // namespace fie

using namespace fie;

extern "C" int fie_block_norm(const fie_norm_args* a, void* stream)
{
    const int rc = norm_check(a);
    if (rc != FIE_OK || a->tokens == 0) return rc;
    hipStream_t st = (hipStream_t)stream;
    hipError_t e = hipSuccess;
    const int64_t most = rows_at_once(a->width);
    for (int64_t row = 0; row < a->tokens && e == hipSuccess; row += most) {
        fie_norm_args part = rows_from(*a, row);
        if (part.tokens > most) part.tokens = most;
        e = norm_run(part, st);
    }
    return launch_status(e, "k_norm");
}
