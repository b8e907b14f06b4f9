/*
 * mako_step.h -- C ABI of the operators around the sampler in a speculative decode step.
 *
 * A step of a serving loop that drafts tokens runs the target model on every request's last token and its drafts, and then
 *
 *   mako_step_cut_rows       what temperature, min_p, top_k and top_p leave of each row of logits: 32 bytes a row, from which
 *                            any token's probability follows (and, where asked for, the row as fp32 probabilities)
 *   mako_step_verify_drafts  accepts drafts against the target's and the drafter's distributions from the caller's uniforms,
 *                            draws the token behind the last accepted one, and gives the requests' new lengths
 *   mako_step_assign_blocks  from those lengths: blocks of a paged cache given back and taken from a free list into block
 *                            tables, and the slot, position and request of every token of the next step
 *
 * all on the device, in stream order, without a trip to the host.  (The reference verifies one draft of a drafter without a
 * distribution, Sampler::verify, src/gen/sampler.cpp:86-107, which mako_sampler.h has bit for bit, for one row per draft; a
 * chain of drafts is its caller's loop, src/gen/session.cpp:481-496.  It has no paged cache.)
 *
 * Every pointer inside a descriptor is a DEVICE pointer.  The calls enqueue their kernels on `stream` (a hipStream_t, or null
 * for the default stream) and return without waiting; they allocate nothing, may be captured into a graph, and leave the
 * calling thread's current device as it was.  One call at a time per context: calls on one context, and replays of graphs
 * that hold such calls, must follow each other in stream order, since they share its scratch memory.  A context outlives the
 * graphs that hold its calls.  Failures are the negative codes of mako_sampler.h; a call that is refused writes nothing, and behind a
 * launch that fails (MAKO_ERR_HIP) nothing more is enqueued and what the call's output arrays hold is undefined, those that replace
 * their inputs too: such a call is repeated from inputs that are known.  Results do not depend on the batch a row is
 * in, nor on timing.
 */
#ifndef MAKO_STEP_H
#define MAKO_STEP_H

#include <stdint.h>

#include "mako_sampler.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Types of logits.  Rows of any element alignment are taken; those at multiples of 16 bytes are read fastest. */
#define MAKO_LOGITS_F32 0u
#define MAKO_LOGITS_BF16 1u
#define MAKO_LOGITS_F16 2u

typedef struct mako_step_ctx mako_step_ctx;

/* Creates a context on HIP device `device` for rows (requests) of up to max_rows and vocabularies of up to max_vocab
 * (at most MAKO_STEP_MAX_ROWS and MAKO_STEP_MAX_VOCAB).  Its scratch memory is allocated here: for every row 160 bytes, 8 for each
 * 1024 of its logits, or part of them, and 32 for each 2048, or 5152 (some 2.5 a logit) with a max_vocab above 6144 (what
 * mako_step_cut_rows writes there: a context that never cuts rows has it too). */
#define MAKO_STEP_MAX_ROWS 65535
#define MAKO_STEP_MAX_VOCAB 1048576
int mako_step_create(mako_step_ctx** out, int device, uint32_t max_rows, uint32_t max_vocab);
void mako_step_destroy(mako_step_ctx* ctx);

/* Text of the last failure on this context (never null). */
const char* mako_step_last_error(const mako_step_ctx* ctx);

/* ---- rows' cuts ----
 * A row's tokens are those that its mask allows and whose logit is neither NaN nor -inf; a logit of +inf counts as the
 * largest finite fp32 number.  (The lowest finite value of a type, which some programs mask with, is a logit like any other:
 * it has a weight of 0 beside an ordinary one, and a row of nothing else is uniform.)  In the order of falling logits, equal
 * ones by token, with the weights exp((logit - max) / temperature), the row keeps
 *   temperature <= 0 (or NaN): the first token alone;  else
 *   min_p > 0:  the tokens whose weight is at least min_p, but at least one; of those
 *   top_k > 0:  the first top_k; of those
 *   top_p < 1:  the least number (at least one) whose weights reach top_p of what all that are left weigh.
 * The filters and their order are the sampler's (src/gen/sampler.cpp:20-62), the penalties are not looked at: there is no
 * history.  Weights and their sums are in 64 bits, where the sampler replays the reference's sums in 32: a cut can differ from
 * the sampler's candidate list by the tokens at its very end.  A weight exp(y) is off by at most 1.6e-14 + 3.4e-16 |y| of itself,
 * a total by at most 1.2e-12 of itself (rows cut to a top_k of 2500; most others by some 1e-14). */
typedef struct mako_row_cut {
    double total;       /* what the kept tokens weigh, the first weighing 1; 0: the row has no token */
    float max_logit;    /* -inf: the row has no token */
    float temperature;  /* the row's; 0 where it is <= 0 or NaN */
    float cut_logit;    /* a token is kept if its logit is above cut_logit, or equal to it and the token <= cut_token; */
    int32_t cut_token;  /* where nothing is cut off: -inf and -1 */
    uint32_t n_kept;
    int32_t top_token;  /* the first token; -1: none */
} mako_row_cut;

typedef struct mako_cut_desc {
    const void* logits;      /* [n_rows][logits_stride] of logits_type; read-only */
    uint32_t logits_type;    /* MAKO_LOGITS_* */
    uint32_t n_rows;
    int64_t logits_stride;   /* elements between rows, >= n_vocab */
    uint32_t n_vocab;
    uint32_t rows_per_params; /* row r has the parameters params[r / rows_per_params]; 0 is 1 */
    const mako_sampling_params* params; /* temperature, top_k, top_p, min_p */
    const uint32_t* mask;    /* optional [n_rows][mask_stride]: bit (i & 31) of word i >> 5 set = token i allowed */
    int64_t mask_stride;     /* 32-bit words between rows, >= ceil(n_vocab / 32) */
    mako_row_cut* out_cuts;  /* [n_rows], 8-byte aligned */
    float* out_probs;        /* optional [n_rows][probs_stride]: weight / total of the kept tokens, 0 for the others; what lies
                                between n_vocab and probs_stride is left as it is */
    int64_t probs_stride;    /* elements between rows, >= n_vocab */
} mako_cut_desc;

int mako_step_cut_rows(mako_step_ctx* ctx, const mako_cut_desc* desc, void* stream);

/* ---- verification of drafts ----
 * Request b has the drafts d_0 .. d_{k-1} (k = n_drafts[b]) and k + 1 rows of the target: row j, the distribution p of the token
 * behind d_{j-1}, is row b * (max_drafts + 1) + j.  The drafter's distribution q that d_j was drawn from is row
 * b * max_drafts + j of `draft`; without `draft`, q is 1 for d_j (a drafter that looks tokens up).  Draft j is accepted if all
 * before it are and u_j q(d_j) < p(d_j) (with probability min(1, p / q)).  Behind the last accepted one a token is drawn by the
 * uniform u[b][max_drafts]: after a rejection from what max(0, p - q) leaves (without `draft`: from p without the draft), else
 * from p; where that leaves nothing, from p.  It is the first whose running sum of weights, in the tokens' order, exceeds the
 * uniform's share of their total.  So tokens are distributed as the target's own are.  A row of p without tokens gives no
 * token (-1); a draft that is no token of the vocabulary is not accepted.
 * Distributions come as logits with their cuts, or, with no cuts, as fp32 probabilities (a value that is not positive and
 * finite is 0).  Sums and comparisons are in 64 bits. */
#define MAKO_STEP_MAX_DRAFTS 64
typedef struct mako_verify_desc {
    uint32_t n_requests;
    uint32_t max_drafts;     /* 0 .. MAKO_STEP_MAX_DRAFTS; 0: every request draws one token from its row */
    uint32_t n_vocab;
    uint32_t target_type;    /* MAKO_LOGITS_*; probabilities are MAKO_LOGITS_F32 */
    const void* target;      /* [n_requests * (max_drafts + 1)][target_stride] */
    int64_t target_stride;   /* elements between rows, >= n_vocab */
    const mako_row_cut* target_cuts; /* of those rows, from mako_step_cut_rows on the same logits and mask; null: the rows
                                are probabilities */
    const uint32_t* target_mask; /* optional, as mako_cut_desc.mask, for logits */
    int64_t target_mask_stride;
    const void* draft;       /* optional [n_requests * max_drafts][draft_stride] */
    uint32_t draft_type;
    uint32_t reserved;       /* 0 */
    int64_t draft_stride;
    const mako_row_cut* draft_cuts;
    const uint32_t* draft_mask;
    int64_t draft_mask_stride;
    const int32_t* draft_tokens; /* [n_requests][max_drafts] */
    const int32_t* n_drafts; /* optional [n_requests], null: max_drafts each; more than max_drafts counts as max_drafts; a
                                request with less than 0 is not there: its outputs are left as they are */
    const float* u;          /* [n_requests][max_drafts + 1] uniforms in [0, 1) */
    const int32_t* seq_len;  /* optional [n_requests]: tokens in the request's cache before this step */
    int32_t* out_tokens;     /* [n_requests][max_drafts + 1]: the accepted drafts, the token drawn, -1 in the other places */
    int32_t* out_accepted;   /* [n_requests]: number of accepted drafts */
    int32_t* out_seq_len;    /* with seq_len, and may be the same array: seq_len + the number of tokens given out.  (The step
                                put the last token and the drafts into the cache; the accepted ones stay.) */
} mako_verify_desc;

int mako_step_verify_drafts(mako_step_ctx* ctx, const mako_verify_desc* desc, void* stream);

/* ---- blocks and slots of a paged cache ----
 * Request b has seq_len[b] tokens in the cache and gets new_len[b] more in the next step; it holds the blocks
 * block_table[b][0 .. n_blocks[b] - 1] of block_size tokens each, and needs w = ceil((seq_len + new_len) / block_size).
 *   1. A request that needs more blocks than a table row has room for (w > max_blocks), or whose positions would pass 31 bits,
 *      gets status MAKO_BLOCKS_WIDE.
 *   2. Blocks beyond w are given back: pushed onto the free list, request by request, in the table's order.
 *   3. Requests that need more blocks take them, in the order of the batch, from the top of the free list, as long as what they
 *      and all such requests before them ask for is there; the others get status MAKO_BLOCKS_SHORT.
 *   4. The new tokens are laid out in the order of the batch: those of request b are the entries out_start[b] to
 *      out_start[b + 1] - 1 of the per-token outputs, as long as those of the request and of all before it that got this far fit
 *      max_tokens; the others get status MAKO_BLOCKS_TOKENS and no blocks (step 3 had counted what they ask for).
 * A request that is refused has no tokens in the step and keeps the blocks that step 2 leaves it.  One that has ended is passed with
 * lengths of 0: it gives all its blocks back.  One with a length below 0 is not there: it keeps its blocks and has no tokens.
 * (A batch of no requests is refused as a whole, where the calls above take one of no rows: there is no out_start to write.)
 * Entries of a table beyond what a request holds are never read, and are left as they are unless blocks are put there.  Blocks
 * are not counted: one that stands in two tables is given back by each. */
#define MAKO_BLOCKS_OK 0
#define MAKO_BLOCKS_SHORT 1
#define MAKO_BLOCKS_WIDE 2
#define MAKO_BLOCKS_TOKENS 3
typedef struct mako_blocks_desc {
    uint32_t n_requests;
    uint32_t block_size;     /* 1 .. 65536 */
    const int32_t* seq_len;  /* [n_requests] */
    const int32_t* new_len;  /* [n_requests] */
    int32_t* block_table;    /* [n_requests][table_stride] */
    int64_t table_stride;    /* entries between rows, >= max_blocks */
    uint32_t max_blocks;
    uint32_t free_capacity;  /* entries of free_blocks: blocks that would be pushed beyond it are lost */
    const int32_t* n_blocks; /* [n_requests] (below 0 counts as 0, above max_blocks as max_blocks) */
    int32_t* out_n_blocks;   /* [n_requests]; may be n_blocks */
    int32_t* free_blocks;    /* [free_capacity]: a stack, the top at n_free - 1 */
    const int32_t* n_free;   /* [1] (below 0 counts as 0, above free_capacity as free_capacity) */
    int32_t* out_n_free;     /* [1]; may be n_free */
    uint32_t max_tokens;     /* entries of the per-token outputs; those behind the last token get slot -1, position 0 and
                                request -1 */
    uint32_t reserved;       /* 0 */
    int32_t* out_start;      /* [n_requests + 1] */
    int32_t* out_status;     /* [n_requests] MAKO_BLOCKS_* */
    int64_t* out_slots;      /* [max_tokens]: block * block_size + place in the block */
    int32_t* out_positions;  /* optional [max_tokens] */
    int32_t* out_request;    /* optional [max_tokens] */
} mako_blocks_desc;

int mako_step_assign_blocks(mako_step_ctx* ctx, const mako_blocks_desc* desc, void* stream);

#ifdef __cplusplus
}
#endif
#endif
