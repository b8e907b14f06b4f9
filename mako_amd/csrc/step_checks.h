// What the step's entry points refuse, before anything is launched (plain C++: host-tested).
#pragma once

#include <stdint.h>

#include "../../include/mako_step.h"

namespace mako {
namespace step {

inline bool type_ok(uint32_t t)
{
    return t == MAKO_LOGITS_F32 || t == MAKO_LOGITS_BF16 || t == MAKO_LOGITS_F16;
}
inline bool aligned(const void* p, uint32_t bytes)
{
    return (reinterpret_cast<uintptr_t>(p) & (bytes - 1u)) == 0;
}
inline bool logits_aligned(const void* p, uint32_t type)
{
    return aligned(p, type == MAKO_LOGITS_F32 ? 4u : 2u);
}
// (null is aligned to anything)
template <class... P>
bool words_aligned(P... p)
{
    return (aligned(p, 4) && ...);
}
inline bool mask_ok(const uint32_t* mask, int64_t stride, uint32_t n_vocab)
{
    return !mask || (aligned(mask, 4) && stride >= (int64_t)(((uint64_t)n_vocab + 31) / 32));
}

// The reason why a context of this size does not take the call, or null.
inline const char* refuse(const mako_cut_desc& d, uint32_t max_rows, uint32_t max_vocab)
{
    if (d.n_vocab == 0)
        return "step: empty vocabulary";
    if (d.n_rows == 0)
        return nullptr;
    if (!d.logits || !d.params || !d.out_cuts)
        return "step: logits, params and out_cuts are required";
    if (d.n_rows > max_rows || d.n_vocab > max_vocab)
        return "step: batch exceeds the context's max_rows/max_vocab";
    if (!type_ok(d.logits_type))
        return "step: unknown type of logits";
    if (!logits_aligned(d.logits, d.logits_type) || !words_aligned(d.params, d.out_probs) || !aligned(d.out_cuts, 8))
        return "step: a pointer is not aligned to its elements (out_cuts: 8 bytes)";
    if (d.logits_stride < (int64_t)d.n_vocab)
        return "step: logits_stride < n_vocab";
    if (!mask_ok(d.mask, d.mask_stride, d.n_vocab))
        return "step: mask_stride < ceil(n_vocab / 32)";
    if (d.out_probs && d.probs_stride < (int64_t)d.n_vocab)
        return "step: probs_stride < n_vocab";
    return nullptr;
}

// The reason why a context of this size does not take the call, or null.
inline const char* refuse(const mako_verify_desc& d, uint32_t max_rows, uint32_t max_vocab)
{
    if (d.n_vocab == 0)
        return "step: empty vocabulary";
    if (d.n_requests == 0)
        return nullptr;
    if (!d.target || !d.u || !d.out_tokens || !d.out_accepted)
        return "step: target, u, out_tokens and out_accepted are required";
    if (d.max_drafts > MAKO_STEP_MAX_DRAFTS)
        return "step: max_drafts > MAKO_STEP_MAX_DRAFTS";
    if (d.max_drafts && !d.draft_tokens)
        return "step: draft_tokens are required";
    if (d.n_requests > max_rows || d.n_vocab > max_vocab)
        return "step: batch exceeds the context's max_rows/max_vocab";
    if (d.reserved)
        return "step: reserved fields are 0";
    if (!type_ok(d.target_type) || (d.draft && !type_ok(d.draft_type)))
        return "step: unknown type of logits";
    if ((!d.target_cuts && d.target_type != MAKO_LOGITS_F32) || (d.draft && !d.draft_cuts && d.draft_type != MAKO_LOGITS_F32))
        return "step: logits need their cuts; probabilities are fp32";
    if ((!d.target_cuts && d.target_mask) || ((!d.draft || !d.draft_cuts) && d.draft_mask))
        return "step: masks go with logits and their cuts";
    if (!d.draft && d.draft_cuts)
        return "step: draft_cuts need draft";
    if (!logits_aligned(d.target, d.target_type) || (d.draft && !logits_aligned(d.draft, d.draft_type)) || !aligned(d.target_cuts, 8) || !aligned(d.draft_cuts, 8) ||
        !words_aligned(d.draft_tokens, d.n_drafts, d.u, d.seq_len, d.out_tokens, d.out_accepted, d.out_seq_len))
        return "step: a pointer is not aligned to its elements (cuts: 8 bytes)";
    if (d.target_stride < (int64_t)d.n_vocab || (d.draft && d.draft_stride < (int64_t)d.n_vocab))
        return "step: target_stride or draft_stride < n_vocab";
    if (!mask_ok(d.target_mask, d.target_mask_stride, d.n_vocab) || !mask_ok(d.draft_mask, d.draft_mask_stride, d.n_vocab))
        return "step: mask_stride < ceil(n_vocab / 32)";
    if ((d.seq_len != nullptr) != (d.out_seq_len != nullptr))
        return "step: seq_len and out_seq_len go together";
    return nullptr;
}

// The reason why a context of this size does not take the call, or null.
inline const char* refuse(const mako_blocks_desc& d, uint32_t max_rows)
{
    if (d.block_size == 0 || d.block_size > 65536)
        return "step: block_size is 1 to 65536";
    if (d.n_requests == 0)
        return "step: no requests";
    if (!d.seq_len || !d.new_len || !d.block_table || !d.n_blocks || !d.out_n_blocks || !d.free_blocks || !d.n_free || !d.out_n_free || !d.out_start || !d.out_status)
        return "step: seq_len, new_len, block_table, n_blocks, free_blocks, n_free, out_start and out_status are required";
    if (d.max_tokens && !d.out_slots)
        return "step: out_slots are required";
    if (d.n_requests > max_rows)
        return "step: batch exceeds the context's max_rows";
    if (d.reserved)
        return "step: reserved fields are 0";
    if (d.max_blocks == 0 || d.table_stride < (int64_t)d.max_blocks)
        return "step: table_stride < max_blocks, or no max_blocks";
    if (d.max_blocks > INT32_MAX || d.free_capacity > INT32_MAX || d.max_tokens > INT32_MAX || (uint64_t)d.n_requests * d.max_blocks > INT32_MAX)
        return "step: blocks and tokens are numbered by 31 bits";
    if (!aligned(d.out_slots, 8) || !words_aligned(d.seq_len, d.new_len, d.block_table, d.n_blocks, d.out_n_blocks, d.free_blocks, d.n_free, d.out_n_free, d.out_start, d.out_status, d.out_positions, d.out_request))
        return "step: a pointer is not aligned to its elements (out_slots: 8 bytes)";
    return nullptr;
}

} // namespace step
} // namespace mako
