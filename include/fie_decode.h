/*
 * fie_decode.h -- C ABI of what a decode step needs around searching and adapters: beam
 * search's selection, states reordered by their parents, pages of a cache, low-rank adapters.
 * No counterpart on the reference's sampler path.
 *
 * Conventions are fie_sampler.h's: device pointers, work enqueued on `stream`, nothing
 * synchronises or allocates, FIE_OK or a negative FIE_E* code, and
 * fie_sampler_last_error() holds the message.
 */
#ifndef FIE_DECODE_H
#define FIE_DECODE_H

#include "fie_ops.h"

#ifdef __cplusplus
extern "C" {
#endif

#define FIE_MAX_BEAMS 64
#define FIE_MAX_EOS 16

/* One step of a beam search over `requests` requests of `beams` beams; row b of request r is
   r * beams + b.  With x the logits (a NaN counts as -inf, +inf as FLT_MAX):
     total[b, v] = scores[b] + ((x[b, v] - m) - log(sum exp(x[b] - m)))      m = max x[b]
   in 64 bits and rounded once to a score, but for the sum: its terms and sums of 32 of them are fp32,
   so its logarithm is off by 2^-24 (6 mean(m - x) + 16) at most, the mean over the terms' weights.
   A request's continuations rank by (total descending, lower beam, larger logit, lower token);
   those of logit -inf do not exist.  Scores and values below -FLT_MAX are held at it, so that none
   is -inf.  The best `beams` that are no eos go on.  An eos continuation among the best `beams` of
   all joins the pool, the request's `beams` best ended ones, at total / (length + 1)^length_penalty;
   on ties the older stays in front.
   Requests that are done, and beams of score -inf, are not read.  A request is done when its
   pool is full and (early_stopping, or the best that goes on is no better than the pool's worst
   at the same length), or when nothing goes on. */
typedef struct fie_beam_args {
    const void* logits;         /* [requests * beams, vocab], rows row_stride elements apart */
    const float* scores;        /* [requests, beams]; -inf: no such beam */
    const int32_t* lengths;     /* [requests] tokens chosen so far */
    const uint8_t* done;        /* [requests] 0 or 1 */
    const float* pool;          /* [requests, beams], -inf where empty */
    const int32_t* ends;        /* [requests, beams, 3]: length, parent row, eos token */
    float* next_scores;         /* these five may be the ones above */
    int32_t* next_lengths;      /* lengths + 1, of requests that were not done */
    uint8_t* next_done;
    float* next_pool;
    int32_t* next_ends;
    int64_t* tokens;            /* [requests * beams]; `pad` where no beam goes on */
    int32_t* parents;           /* [requests * beams] rows; the row itself where none goes on */
    int32_t* history_tokens;    /* [history_steps, requests * beams], or NULL: the step's tokens and */
    int32_t* history_parents;   /* parents are kept at [lengths[r]] too */
    int64_t row_stride;
    void* workspace;            /* fie_beam_workspace_size() bytes, 16-byte aligned */
    size_t workspace_bytes;
    double length_penalty;
    int32_t requests, beams, vocab, dtype;
    int32_t early_stopping, min_tokens, pad, history_steps;   /* before min_tokens no eos exists */
    int32_t eos_count;
    int32_t eos[FIE_MAX_EOS];
    int32_t max_tokens;         /* continuations of so many tokens end, whatever their token; 0: none */
} fie_beam_args;

size_t fie_beam_workspace_size(const fie_beam_args* args);

int fie_beam_step(const fie_beam_args* args, void* stream);

/* Rows of up to FIE_MAX_STATES tensors gathered: dst row i is src row parents[i]; a parent
   outside [0, rows) stands for i.  Outputs have no memory of any input or each other.  One call takes fewer
   than 2^24 pieces of 16 KB, a row of each tensor at least one. */
#define FIE_MAX_STATES 48
typedef struct fie_state {
    const void* src;            /* [rows], row_bytes each, src_stride bytes apart */
    void* dst;                  /* [n] likewise, n <= rows */
    int64_t src_stride, dst_stride, row_bytes, rows;
} fie_state;

typedef struct fie_states_args {
    const int32_t* parents;     /* [n] */
    int32_t n, count;           /* rows that are written; tensors */
    fie_state state[FIE_MAX_STATES];        /* those past count need not be there */
} fie_states_args;

int fie_reorder_states(const fie_states_args* args, void* stream);

/* Pages of a cache: `rows` sequences, each with up to `wide` pages of `page` tokens out of a pool
   of `pages`.  A page may be in several rows' tables, always at the same place of a row.
   The state is one array of int32 (fie_pages_state_ints):
     table  [rows][wide]    page ids, -1 past a row's pages
     lengths [rows]         tokens
     refs   [pages]         table entries that hold the page; 0: free
     blocks [ceil(pages / 1024)]   free pages among each 1024
   The scratch (fie_pages_scratch_bytes, 16-byte aligned) holds nothing between calls. */
#define FIE_MAX_PAGE_ROWS 4096
#define FIE_MAX_PAGES (1 << 21)

/* Cache tensors of one layout: a page is `outer` pieces, outer_stride bytes apart, of `page`
   tokens of token_bytes one after another; with `whole` of token_bytes that go with the whole page. */
typedef struct fie_cache_group {
    void* const* base;          /* [count] on the device */
    int64_t page_stride, outer_stride, token_bytes;
    int32_t count, outer, whole;
    int32_t shift;              /* 0: every base and stride is a multiple of 16 */
} fie_cache_group;

#define FIE_MAX_CACHE_GROUPS 8
typedef struct fie_pages_args {
    int32_t* state;
    void* scratch;
    size_t scratch_bytes;
    int32_t pages, page, rows, wide;
    const int32_t* parents;     /* [rows] or NULL: each its own; outside [0, rows): the row is emptied */
    const int32_t* lengths;     /* [rows] or NULL: its parent's */
    uint8_t* granted;           /* [rows]: 0 where pages did not suffice */
    int32_t* live;              /* fie_pages_compact: pages in use */
    const int32_t* src;         /* fie_pages_copy: [copies] pages */
    const int32_t* dst;
    int32_t copies, group_count;
    fie_cache_group group[FIE_MAX_CACHE_GROUPS];
} fie_pages_args;

size_t fie_pages_state_ints(int32_t pages, int32_t rows, int32_t wide);
size_t fie_pages_scratch_bytes(int32_t pages, int32_t rows);

/* Row i takes its parent's pages, as many as min(lengths[i], the parent's length) tokens need;
   what no row holds any more is free.  Where lengths[i] is more, the row grows to it, in the rows'
   order and by the lowest free pages; a last page that is not full and that other rows hold is
   replaced by a copy first, but for the longest (then lowest) row where all its holders grow.  A
   row whose pages, with those of the rows before it, are more than are free, or more than `wide`,
   does not grow. */
int fie_pages_step(const fie_pages_args* args, void* stream);

/* The i-th used page at or past the count of used pages moves to the i-th free page below it. */
int fie_pages_compact(const fie_pages_args* args, void* stream);

/* Pages dst[i] become copies of src[i] (those outside [0, pages) are left out); no table changes. */
int fie_pages_copy(const fie_pages_args* args, void* stream);

/* Low-rank adapters of many tokens: with i = ids[t],
     y[t] = base[t] + scale[i] * b[i] (a[i] x[t])          (ids[t] outside [0, adapters): base[t])
   Products of x and a are exact and their sums fp32.  With fp16 and bf16 adapters each number of
   a[i] x[t] enters the second product as the sum of two of their type, off by 2^-16 of itself (bf16) or
   by 2^-22 of itself or 2^-39 of the token's largest, whichever is more (fp16); that product's sums are
   fp32, and y is rounded once.  An adapter of rank 0 gives base.
   Infinite and NaN numbers of x give what the formula gives, for their token alone; those of a and b are
   for the adapter's tokens NaN as a rule. */
#define FIE_MAX_RANK 256
#define FIE_MAX_ADAPTERS 4096
#define FIE_ADAPTER_K 64        /* rows of a are padded with zeros to a multiple of so many */
#define FIE_ADAPTER_RANK 16     /* ranks likewise, in a and b */

/* Whose tokens are whose: tokens by adapter, in tiles of up to 16.  plan is
   fie_adapter_plan_ints() of int32. */
typedef struct fie_adapter_plan_args {
    const int32_t* ids;         /* [tokens] */
    int32_t* plan;
    int32_t tokens, adapters;
} fie_adapter_plan_args;

size_t fie_adapter_plan_ints(int32_t tokens, int32_t adapters);
int fie_adapter_plan(const fie_adapter_plan_args* args, void* stream);

typedef struct fie_adapter_args {
    const void* x;              /* [tokens, k] in dtype, or int8 with x_scale */
    const float* x_scale;       /* [tokens] */
    const void* a;              /* [adapters, rank, k_pad], zeros past each adapter's rank and past k */
    const void* b;              /* [adapters, n, rank], likewise, b_pitch elements between channels */
    const float* scale;         /* [adapters] */
    const int32_t* ranks;       /* [adapters], 0..rank */
    const int32_t* plan;        /* of these tokens and so many adapters */
    const void* base;           /* [tokens, n] in y_dtype or fp32, or NULL: 0; may be y */
    void* y;                    /* [tokens, n] */
    void* workspace;            /* fie_adapter_workspace_size() bytes, 16-byte aligned */
    size_t workspace_bytes;
    int64_t x_stride, base_stride, y_stride;        /* elements between rows */
    int32_t tokens, k, n, adapters;
    int32_t rank, k_pad;        /* rank a multiple of FIE_ADAPTER_RANK, k_pad of FIE_ADAPTER_K */
    int32_t b_pitch;            /* rank or more; a multiple of 16 bytes, best none of 128 */
    int32_t dtype, x_dtype;     /* the adapters' type; x's: that or FIE_I8 */
    int32_t y_dtype, base_dtype;        /* dtype or FIE_F32; y_dtype or FIE_F32 */
    int32_t reserved;
} fie_adapter_args;

size_t fie_adapter_workspace_size(const fie_adapter_args* args);
int fie_adapter_linear(const fie_adapter_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FIE_DECODE_H */
