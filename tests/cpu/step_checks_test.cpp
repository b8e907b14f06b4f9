// What the step's entry points refuse (mako_amd/csrc/step_checks.h), without a GPU: every refused field once, on top of a call
// that is taken.
#include <stdio.h>
#include <string.h>

#include "../../mako_amd/csrc/step_checks.h"

using mako::step::refuse;

static int failures = 0;

static void expect(const char* name, const char* got, const char* part)
{
    const bool ok = part ? got && strstr(got, part) : !got;
    if (!ok) {
        printf("%s: got %s, expected %s\n", name, got ? got : "(taken)", part ? part : "(taken)");
        ++failures;
    }
}

template <class T>
static T* at(uintptr_t a)
{
    return reinterpret_cast<T*>(a);
}

int main()
{
    const uint32_t rows = 64, vocab = 1000;
    mako_cut_desc c;
    memset(&c, 0, sizeof c);
    c.logits = at<void>(4096);
    c.logits_type = MAKO_LOGITS_BF16;
    c.n_rows = 64;
    c.n_vocab = 1000;
    c.logits_stride = 1000;
    c.params = at<mako_sampling_params>(4096);
    c.out_cuts = at<mako_row_cut>(4096);
#define CUT(change, part)                                                                                          \
    do {                                                                                                           \
        mako_cut_desc d = c;                                                                                       \
        change;                                                                                                    \
        expect("cut: " #change, refuse(d, rows, vocab), part);                                                     \
    } while (0)
    CUT(, nullptr);
    CUT(d.n_vocab = 0, "empty vocabulary");
    CUT(d.n_rows = 0; d.logits = nullptr, nullptr);
    CUT(d.logits = nullptr, "required");
    CUT(d.params = nullptr, "required");
    CUT(d.out_cuts = nullptr, "required");
    CUT(d.n_rows = 65, "max_rows");
    CUT(d.n_vocab = 1001; d.logits_stride = 1001, "max_vocab");
    CUT(d.logits_type = 3, "type");
    CUT(d.logits = at<void>(4098), nullptr);
    CUT(d.logits = at<void>(4097), "aligned");
    CUT(d.logits = at<void>(4098); d.logits_type = MAKO_LOGITS_F32, "aligned");
    CUT(d.params = at<mako_sampling_params>(4098), "aligned");
    CUT(d.out_cuts = at<mako_row_cut>(4100), "aligned");
    CUT(d.logits_stride = 999, "logits_stride");
    CUT(d.logits_stride = -1000, "logits_stride");
    CUT(d.mask = at<uint32_t>(4096); d.mask_stride = 32, nullptr);
    CUT(d.mask = at<uint32_t>(4096); d.mask_stride = 31, "mask");
    CUT(d.mask = at<uint32_t>(4097); d.mask_stride = 32, "mask");
    CUT(d.out_probs = at<float>(4096); d.probs_stride = 1000, nullptr);
    CUT(d.out_probs = at<float>(4096); d.probs_stride = 999, "probs_stride");
    CUT(d.out_probs = at<float>(4097); d.probs_stride = 1000, "aligned");

    mako_verify_desc v;
    memset(&v, 0, sizeof v);
    v.n_requests = 64;
    v.max_drafts = 4;
    v.n_vocab = 1000;
    v.target = at<void>(4096);
    v.target_type = MAKO_LOGITS_F16;
    v.target_stride = 1000;
    v.target_cuts = at<mako_row_cut>(4096);
    v.draft_tokens = at<int32_t>(4096);
    v.u = at<float>(4096);
    v.out_tokens = at<int32_t>(4096);
    v.out_accepted = at<int32_t>(4096);
#define VERIFY(change, part)                                                                                       \
    do {                                                                                                           \
        mako_verify_desc d = v;                                                                                    \
        change;                                                                                                    \
        expect("verify: " #change, refuse(d, rows, vocab), part);                                                  \
    } while (0)
#define DRAFT d.draft = at<void>(4096); d.draft_type = MAKO_LOGITS_BF16; d.draft_stride = 1000; d.draft_cuts = at<mako_row_cut>(4096)
    VERIFY(, nullptr);
    VERIFY(DRAFT, nullptr);
    VERIFY(DRAFT; d.draft_type = MAKO_LOGITS_F32; d.draft_cuts = nullptr, nullptr);
    VERIFY(d.target_type = MAKO_LOGITS_F32; d.target_cuts = nullptr, nullptr);
    VERIFY(d.n_requests = 0; d.target = nullptr, nullptr);
    VERIFY(d.n_vocab = 0, "empty vocabulary");
    VERIFY(d.target = nullptr, "required");
    VERIFY(d.u = nullptr, "required");
    VERIFY(d.out_tokens = nullptr, "required");
    VERIFY(d.out_accepted = nullptr, "required");
    VERIFY(d.max_drafts = 64, nullptr);
    VERIFY(d.max_drafts = 65, "MAX_DRAFTS");
    VERIFY(d.draft_tokens = nullptr, "draft_tokens");
    VERIFY(d.max_drafts = 0; d.draft_tokens = nullptr, nullptr);
    VERIFY(d.n_requests = 65, "max_rows");
    VERIFY(d.n_vocab = 1001; d.target_stride = 1001, "max_vocab");
    VERIFY(d.reserved = 1, "reserved");
    VERIFY(d.target_type = 9, "type");
    VERIFY(DRAFT; d.draft_type = 9, "type");
    VERIFY(d.target_cuts = nullptr, "probabilities are fp32");
    VERIFY(DRAFT; d.draft_cuts = nullptr, "probabilities are fp32");
    VERIFY(d.target_type = MAKO_LOGITS_F32; d.target_cuts = nullptr; d.target_mask = at<uint32_t>(4096); d.target_mask_stride = 32, "masks go with logits");
    VERIFY(d.draft_mask = at<uint32_t>(4096); d.draft_mask_stride = 32, "masks go with logits");
    VERIFY(d.draft_cuts = at<mako_row_cut>(4096), "need draft");
    VERIFY(d.target = at<void>(4097), "aligned");
    VERIFY(DRAFT; d.draft = at<void>(4097), "aligned");
    VERIFY(d.target_cuts = at<mako_row_cut>(4100), "aligned");
    VERIFY(d.u = at<float>(4098), "aligned");
    VERIFY(d.out_tokens = at<int32_t>(4097), "aligned");
    VERIFY(d.target_stride = 999, "stride");
    VERIFY(DRAFT; d.draft_stride = 999, "stride");
    VERIFY(d.target_mask = at<uint32_t>(4096); d.target_mask_stride = 31, "mask_stride");
    VERIFY(DRAFT; d.draft_mask = at<uint32_t>(4096); d.draft_mask_stride = 31, "mask_stride");
    VERIFY(d.seq_len = at<int32_t>(4096), "go together");
    VERIFY(d.out_seq_len = at<int32_t>(4096), "go together");
    VERIFY(d.seq_len = at<int32_t>(4096); d.out_seq_len = at<int32_t>(4096), nullptr);

    mako_blocks_desc b;
    memset(&b, 0, sizeof b);
    b.n_requests = 64;
    b.block_size = 16;
    b.seq_len = b.new_len = b.n_blocks = b.n_free = at<int32_t>(4096);
    b.block_table = b.out_n_blocks = b.free_blocks = b.out_n_free = b.out_start = b.out_status = at<int32_t>(4096);
    b.table_stride = 100;
    b.max_blocks = 100;
    b.free_capacity = 1000;
    b.max_tokens = 128;
    b.out_slots = at<int64_t>(4096);
#define BLOCKS(change, part)                                                                                       \
    do {                                                                                                           \
        mako_blocks_desc d = b;                                                                                    \
        change;                                                                                                    \
        expect("blocks: " #change, refuse(d, rows), part);                                                         \
    } while (0)
    BLOCKS(, nullptr);
    BLOCKS(d.block_size = 0, "block_size");
    BLOCKS(d.block_size = 65537, "block_size");
    BLOCKS(d.n_requests = 0, "no requests");
    BLOCKS(d.n_requests = 65, "max_rows");
    BLOCKS(d.seq_len = nullptr, "required");
    BLOCKS(d.new_len = nullptr, "required");
    BLOCKS(d.block_table = nullptr, "required");
    BLOCKS(d.n_blocks = nullptr, "required");
    BLOCKS(d.out_n_blocks = nullptr, "required");
    BLOCKS(d.free_blocks = nullptr, "required");
    BLOCKS(d.n_free = nullptr, "required");
    BLOCKS(d.out_n_free = nullptr, "required");
    BLOCKS(d.out_start = nullptr, "required");
    BLOCKS(d.out_status = nullptr, "required");
    BLOCKS(d.out_slots = nullptr, "out_slots");
    BLOCKS(d.out_slots = nullptr; d.max_tokens = 0, nullptr);
    BLOCKS(d.reserved = 1, "reserved");
    BLOCKS(d.max_blocks = 0, "max_blocks");
    BLOCKS(d.table_stride = 99, "table_stride");
    BLOCKS(d.max_blocks = 0x80000000u; d.table_stride = 0x80000000ll, "31 bits");
    BLOCKS(d.max_blocks = 40000000u; d.table_stride = 40000000, "31 bits");
    BLOCKS(d.free_capacity = 0x80000000u, "31 bits");
    BLOCKS(d.max_tokens = 0x80000000u, "31 bits");
    BLOCKS(d.out_slots = at<int64_t>(4100), "aligned");
    BLOCKS(d.block_table = at<int32_t>(4098), "aligned");
    BLOCKS(d.out_positions = at<int32_t>(4097), "aligned");
    if (!failures)
        printf("ok\n");
    return failures ? 1 : 0;
}
