// C ABI of include/mako_step.h over the kernels of k_step_cut.hip, k_step_verify.hip and k_step_blocks.hip.
#include <hip/hip_runtime.h>

#include <stdint.h>
#include <stdio.h>

#include <new>

#include "../../include/mako_step.h"
#include "step_checks.h"
#include "step_common.h"
#include "step_cut.h"
#include "step_launch.h"

struct mako_step_ctx {
    int device = 0;
    uint32_t max_rows = 0, max_vocab = 0;
    mako::step::Scratch sc{};
    char err[192] = "";
};

namespace {

// The context's device for the length of a call; the thread's own again behind it.
class OnDevice {
public:
    explicit OnDevice(int device)
    {
        status_ = hipGetDevice(&before_);
        if (status_ == hipSuccess && before_ != device) {
            status_ = hipSetDevice(device);
            moved_ = status_ == hipSuccess;
        }
    }
    ~OnDevice()
    {
        if (moved_)
            (void)hipSetDevice(before_);
    }
    hipError_t status() const { return status_; }

private:
    int before_ = 0;
    bool moved_ = false;
    hipError_t status_;
};

int fail(mako_step_ctx* ctx, int code, const char* what, const char* more = "")
{
    snprintf(ctx->err, sizeof ctx->err, "%s%s", what, more);
    return code;
}
// Of a call's launches (by their own statuses: an error that an earlier call left is that call's, and stays; a failed launch is
// reported by this call, not by the next that looks).
int launched(mako_step_ctx* ctx, hipError_t e)
{
    if (e == hipSuccess)
        return MAKO_OK;
    (void)hipGetLastError();
    return fail(ctx, MAKO_ERR_HIP, "step: a kernel could not be launched: ", hipGetErrorString(e));
}

template <class T>
hipError_t take(T*& p, uint64_t count)
{
    return hipMalloc(reinterpret_cast<void**>(&p), count * sizeof(T));
}

} // namespace

extern "C" {

int mako_step_create(mako_step_ctx** out, int device, uint32_t max_rows, uint32_t max_vocab)
{
    if (!out)
        return MAKO_ERR_INVALID_ARG;
    *out = nullptr;
    if (max_rows == 0 || max_vocab == 0 || max_rows > MAKO_STEP_MAX_ROWS || max_vocab > MAKO_STEP_MAX_VOCAB)
        return MAKO_ERR_INVALID_ARG;
    mako_step_ctx* ctx = new (std::nothrow) mako_step_ctx;
    if (!ctx)
        return MAKO_ERR_NO_MEMORY;
    ctx->device = device;
    ctx->max_rows = max_rows;
    ctx->max_vocab = max_vocab;
    const OnDevice on(device);
    mako::step::Scratch& sc = ctx->sc;
    sc.chunks_cap = mako::step::chunks_of(max_vocab);
    sc.parts_cap = (max_vocab + mako::step::kPart - 1) / mako::step::kPart;
    const uint64_t rows = max_rows;
    hipError_t e = on.status();
    if (e == hipSuccess)
        e = take(sc.chunks, rows * sc.chunks_cap);
    const bool lists = max_vocab > mako::step::kWholeRow; // (rows that are held whole have none)
    if (e == hipSuccess && lists)
        e = take(sc.lists, rows * sc.chunks_cap * mako::step::kChunkList);
    if (e == hipSuccess && lists)
        e = take(sc.looks, rows * sc.chunks_cap * mako::step::kLookList);
    if (e == hipSuccess)
        e = take(sc.plans, rows);
    if (e == hipSuccess)
        e = take(sc.wide, 1);
    if (e == hipSuccess)
        e = take(sc.parts, rows * sc.parts_cap);
    if (e == hipSuccess)
        e = take(sc.stops, rows);
    if (e == hipSuccess)
        e = take(sc.released, rows + 1);
    if (e == hipSuccess)
        e = take(sc.taken, rows + 1);
    if (e == hipSuccess)
        e = take(sc.held, rows);
    if (e == hipSuccess)
        e = take(sc.start, rows + 1);
    if (e == hipSuccess)
        e = take(sc.free_state, 2);
    if (e == hipSuccess)
        e = mako::step::init_cut();
    if (e != hipSuccess) {
        (void)hipGetLastError();
        mako_step_destroy(ctx);
        return e == hipErrorOutOfMemory ? MAKO_ERR_NO_MEMORY : MAKO_ERR_HIP;
    }
    *out = ctx;
    return MAKO_OK;
}

void mako_step_destroy(mako_step_ctx* ctx)
{
    if (!ctx)
        return;
    {
        const OnDevice on(ctx->device);
        mako::step::Scratch& sc = ctx->sc;
        void* ptrs[] = {sc.chunks, sc.lists, sc.looks, sc.plans, sc.wide, sc.parts, sc.stops, sc.released, sc.taken, sc.held, sc.start, sc.free_state};
        for (void* p : ptrs)
            if (p)
                (void)hipFree(p);
    }
    delete ctx;
}

const char* mako_step_last_error(const mako_step_ctx* ctx)
{
    return ctx ? ctx->err : "null context";
}

int mako_step_cut_rows(mako_step_ctx* ctx, const mako_cut_desc* desc, void* stream)
{
    if (!ctx || !desc)
        return MAKO_ERR_INVALID_ARG;
    mako_cut_desc d = *desc;
    if (const char* why = mako::step::refuse(d, ctx->max_rows, ctx->max_vocab))
        return fail(ctx, MAKO_ERR_INVALID_ARG, why);
    if (d.n_rows == 0)
        return MAKO_OK;
    if (d.rows_per_params == 0)
        d.rows_per_params = 1;
    const OnDevice on(ctx->device);
    if (on.status() != hipSuccess)
        return fail(ctx, MAKO_ERR_HIP, "step: the context's device: ", hipGetErrorString(on.status()));
    hipStream_t st = static_cast<hipStream_t>(stream);
    hipError_t e = mako::step::launch_cut(st, d, ctx->sc);
    if (e == hipSuccess && d.out_probs)
        e = mako::step::launch_probs(st, d);
    return launched(ctx, e);
}

int mako_step_verify_drafts(mako_step_ctx* ctx, const mako_verify_desc* desc, void* stream)
{
    if (!ctx || !desc)
        return MAKO_ERR_INVALID_ARG;
    const mako_verify_desc& d = *desc;
    if (const char* why = mako::step::refuse(d, ctx->max_rows, ctx->max_vocab))
        return fail(ctx, MAKO_ERR_INVALID_ARG, why);
    if (d.n_requests == 0)
        return MAKO_OK;
    const OnDevice on(ctx->device);
    if (on.status() != hipSuccess)
        return fail(ctx, MAKO_ERR_HIP, "step: the context's device: ", hipGetErrorString(on.status()));
    return launched(ctx, mako::step::launch_verify(static_cast<hipStream_t>(stream), d, ctx->sc));
}

int mako_step_assign_blocks(mako_step_ctx* ctx, const mako_blocks_desc* desc, void* stream)
{
    if (!ctx || !desc)
        return MAKO_ERR_INVALID_ARG;
    const mako_blocks_desc& d = *desc;
    if (const char* why = mako::step::refuse(d, ctx->max_rows))
        return fail(ctx, MAKO_ERR_INVALID_ARG, why);
    const OnDevice on(ctx->device);
    if (on.status() != hipSuccess)
        return fail(ctx, MAKO_ERR_HIP, "step: the context's device: ", hipGetErrorString(on.status()));
    return launched(ctx, mako::step::launch_blocks(static_cast<hipStream_t>(stream), d, ctx->sc));
}

} // extern "C"
