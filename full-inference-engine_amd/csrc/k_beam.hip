// Beam search's selection behind the C ABI of include/fie_decode.h.
#include <algorithm>
#include <cmath>

#include "beam.h"
#include "states.h"

namespace fie {

static BeamWork beam_work(const fie_beam_args& a)
{
    BeamWork w;
    const int rows = a.requests * a.beams;
    // 7 elements more: rows need not begin at 16 bytes
    const int tiles = (a.vocab + 7 + kBeamTile - 1) / kBeamTile;
    // as many workgroups as the CUs hold at a time, each with one long span: the rest would be a second
    // round of few
    const int hold = (a.dtype == FIE_BF16 ? kBeamHold<FIE_BF16> : kBeamHold<FIE_F32>) * std::max(cu_count(), 1);
    const int spans = std::min({kBeamSpans, tiles, std::max(1, hold / std::max(rows, 1))});
    w.tiles = (tiles + spans - 1) / spans;
    w.spans = (tiles + w.tiles - 1) / w.tiles;
    w.most = std::min(a.vocab, a.beams + a.eos_count);
    w.span = (BeamSpan*)a.workspace;
    w.cand = (uint64_t*)(w.span + (int64_t)rows * w.spans);
    return w;
}

static size_t beam_bytes(const fie_beam_args& a)
{
    const BeamWork w = beam_work(a);
    return (size_t)a.requests * a.beams * w.spans * (sizeof(BeamSpan) + 8 * (size_t)w.most);
}

static hipError_t beam_run(const fie_beam_args& a, hipStream_t st)
{
    const BeamWork w = beam_work(a);
    const int rows = a.requests * a.beams;
    const dim3 grid((unsigned)w.spans, (unsigned)rows);
    switch (a.dtype) {
    case FIE_F32: k_beam_scan<FIE_F32><<<grid, kBeamThreads, 0, st>>>(a, w); break;
    case FIE_F16: k_beam_scan<FIE_F16><<<grid, kBeamThreads, 0, st>>>(a, w); break;
    default: k_beam_scan<FIE_BF16><<<grid, kBeamThreads, 0, st>>>(a, w); break;
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    // all candidates of a request at once, or, where there are many, a wave a row as far as the spans'
    // lists fit
    const int all = a.beams * w.spans * w.most, wanted = a.beams * (1 + a.eos_count);
    const size_t lists = (size_t)w.spans * w.most * 8, own = (size_t)a.beams * w.most * 8;
    const bool ranked = all <= 1024 * kPickEach && wanted <= kPickList / 4;
    const int fits = (int)std::max<size_t>(2, (((size_t)140 << 10) - own) / lists);
    const int waves = std::min(fits, (ranked ? std::max(4, std::min(15, (all + 127) / 128)) : std::min(a.beams, 15)) + beam_power(a.length_penalty));
    const bool at_once = ranked && all <= 64 * waves * kPickEach;
    const size_t lds = std::max(waves * lists + own, at_once ? (size_t)kPickList * 32 : 0);
    k_beam_pick<<<(unsigned)a.requests, 64 * waves, lds, st>>>(a, w, at_once ? wanted : 0);
    return hipGetLastError();
}

static int beam_sizes(const fie_beam_args* a)
{
    if (a->beams < 1 || a->beams > FIE_MAX_BEAMS) return fail(FIE_E_ARG, "beams out of range [1, 64]");
    if (a->requests < 0 || (int64_t)a->requests * a->beams > 65535) return fail(FIE_E_ARG, "more than 65535 rows");
    if (a->vocab < 1 || a->vocab > kMaxTiles * kTile) return fail(FIE_E_ARG, "vocab out of range [1, 524288]");
    if (a->dtype < FIE_F32 || a->dtype > FIE_BF16) return fail(FIE_E_ARG, "unknown dtype");
    if (a->eos_count < 0 || a->eos_count > FIE_MAX_EOS) return fail(FIE_E_ARG, "eos_count out of range [0, 16]");
    return FIE_OK;
}

static int beam_check(const fie_beam_args* a)
{
    if (!a) return fail(FIE_E_ARG, "args is NULL");
    if (const int rc = beam_sizes(a); rc != FIE_OK) return rc;
    if (a->row_stride < a->vocab) return fail(FIE_E_ARG, "row_stride < vocab");
    if (!std::isfinite(a->length_penalty)) return fail(FIE_E_ARG, "length_penalty is not finite");
    if (a->requests == 0) return FIE_OK;
    if (!a->logits || !a->scores || !a->lengths || !a->done || !a->pool || !a->ends || !a->next_scores || !a->next_lengths ||
        !a->next_done || !a->next_pool || !a->next_ends || !a->tokens || !a->parents)
        return fail(FIE_E_ARG, "a required pointer is NULL");
    if ((uintptr_t)a->logits % (a->dtype == FIE_F32 ? 4 : 2)) return fail(FIE_E_ARG, "logits are not aligned to their type");
    if (a->max_tokens < 0 || a->min_tokens < 0) return fail(FIE_E_ARG, "min_tokens or max_tokens < 0");
    if (!a->history_tokens != !a->history_parents || a->history_steps < 0)
        return fail(FIE_E_ARG, "a history is tokens and parents of a number of steps");
    if (!a->workspace || a->workspace_bytes < beam_bytes(*a)) return fail(FIE_E_WORKSPACE, "workspace too small");
    if (((uintptr_t)a->workspace & 15) != 0) return fail(FIE_E_WORKSPACE, "workspace not 16-byte aligned");
    return FIE_OK;
}

}  // namespace fie

using namespace fie;

extern "C" size_t fie_beam_workspace_size(const fie_beam_args* a)
{
    return a && a->requests > 0 && beam_sizes(a) == FIE_OK ? beam_bytes(*a) : 0;
}

extern "C" int fie_beam_step(const fie_beam_args* a, void* stream)
{
    const int rc = beam_check(a);
    if (rc != FIE_OK || a->requests == 0) return rc;
    return launch_status(beam_run(*a, (hipStream_t)stream), "k_beam");
}

extern "C" int fie_reorder_states(const fie_states_args* a, void* stream)
{
    if (!a) return fail(FIE_E_ARG, "args is NULL");
    if (a->n < 0 || a->count < 0 || a->count > FIE_MAX_STATES) return fail(FIE_E_ARG, "n or count out of range");
    if (a->n == 0 || a->count == 0) return FIE_OK;
    if (!a->parents) return fail(FIE_E_ARG, "parents is NULL");
    fie_states_args held;               // entries past count need not be there
    held.parents = a->parents;
    held.n = a->n;
    held.count = a->count;
    StateBlocks b;
    int64_t blocks = 0;
    for (int i = 0; i < a->count; ++i) {
        const fie_state& s = a->state[i];
        if (!s.src || !s.dst) return fail(FIE_E_ARG, "a state is NULL");
        if (s.rows < a->n || s.row_bytes < 1 || s.row_bytes > INT64_C(1) << 40) return fail(FIE_E_ARG, "a state's rows are fewer than n, or empty");
        if (a->n > 1 && s.dst_stride < s.row_bytes) return fail(FIE_E_ARG, "output rows overlap");
        b.chunks[i] = (int32_t)((s.row_bytes + 15 + kCopyChunk - 1) / kCopyChunk);
        blocks += (int64_t)b.chunks[i] * a->n;
        if (blocks > kMostBlocks) return fail(FIE_E_ARG, "more than one launch holds");
        b.end[i] = (int32_t)blocks;
        held.state[i] = s;
    }
    k_reorder<<<(unsigned)blocks, kCopyThreads, 0, (hipStream_t)stream>>>(held, b);
    return launch_status(hipGetLastError(), "k_reorder");
}
