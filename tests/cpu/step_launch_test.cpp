// What the step's entry points do where launches fail, without a GPU: the HIP functions that they call are this program's (its
// symbols come before the runtime's), and count the launches.
#include <dlfcn.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <utility>

#include "../../include/mako_step.h"

namespace {
struct Dim {
    uint32_t x, y, z;
};
constexpr int kNotReady = 600, kOutOfResources = 701; // hipErrorNotReady, hipErrorLaunchOutOfResources
int pending = 0;  // the thread's last error
int launches = 0, failing = 0; // the launch that fails, from 1 on
uint64_t allocated = 0, most = ~0ull; // bytes, and how many there are
int failures = 0;

void expect(const char* call, const char* what, bool ok)
{
    if (!ok) {
        printf("%s: %s\n", call, what);
        ++failures;
    }
}
} // namespace

extern "C" {
int hipGetDevice(int* device)
{
    *device = 0;
    return 0;
}
int hipSetDevice(int)
{
    return 0;
}
int hipMalloc(void** p, size_t bytes)
{
    *p = bytes <= most - allocated ? malloc(bytes) : nullptr;
    allocated += *p ? bytes : 0;
    return *p ? 0 : pending = 2; // hipErrorOutOfMemory
}
int hipFree(void* p)
{
    free(p);
    return 0;
}
int hipFuncSetAttribute(const void*, int, int)
{
    return 0;
}
int hipGetLastError()
{
    const int e = pending;
    pending = 0;
    return e;
}
int __hipPushCallConfiguration(Dim, Dim, size_t, void*)
{
    return 0;
}
int __hipPopCallConfiguration(Dim* grid, Dim* block, size_t* lds, void** stream)
{
    *grid = *block = {1, 1, 1};
    *lds = 0;
    *stream = nullptr;
    return 0;
}
int hipLaunchKernel(const void*, Dim, Dim, void**, size_t, void*)
{
    return ++launches == failing ? pending = kOutOfResources : 0;
}
}

int main(int, char** argv)
{
    void* lib = dlopen(argv[1], RTLD_NOW | RTLD_LOCAL);
    if (!lib) {
        printf("%s\n", dlerror());
        return 1;
    }
    const auto create = reinterpret_cast<decltype(&mako_step_create)>(dlsym(lib, "mako_step_create"));
    const auto destroy = reinterpret_cast<decltype(&mako_step_destroy)>(dlsym(lib, "mako_step_destroy"));
    const auto cut_rows = reinterpret_cast<decltype(&mako_step_cut_rows)>(dlsym(lib, "mako_step_cut_rows"));
    const auto verify_drafts = reinterpret_cast<decltype(&mako_step_verify_drafts)>(dlsym(lib, "mako_step_verify_drafts"));
    const auto last_error = reinterpret_cast<decltype(&mako_step_last_error)>(dlsym(lib, "mako_step_last_error"));
    const auto assign_blocks = reinterpret_cast<decltype(&mako_step_assign_blocks)>(dlsym(lib, "mako_step_assign_blocks"));
    mako_step_ctx* ctx = nullptr;
    // a context's memory is what the header says, whole or not at all
    const auto parts = [](uint64_t vocab, uint64_t of) { return (vocab + of - 1) / of; };
    for (const auto& size : {std::pair<uint32_t, uint32_t>{65535, 1}, {65535, 6144}, {3, 6145}, {500, 129280}, {1, 1048576}}) {
        const uint64_t rows = size.first, bytes = rows * (160 + parts(size.second, 1024) * 8 + parts(size.second, 2048) * (size.second > 6144 ? 5152 : 32));
        char name[64];
        snprintf(name, sizeof name, "context for %u rows of %u", size.first, size.second);
        allocated = 0;
        expect(name, "fails", create(&ctx, 0, size.first, size.second) == MAKO_OK && ctx);
        if (allocated < bytes || allocated > bytes + 64) // (a few words of the batch)
            printf("%llu bytes, expected %llu\n", (unsigned long long)allocated, (unsigned long long)bytes);
        expect(name, "memory", allocated >= bytes && allocated <= bytes + 64);
        destroy(ctx);
        allocated = 0;
        most = bytes - 1;
        expect(name, "with too little memory", create(&ctx, 0, size.first, size.second) == MAKO_ERR_NO_MEMORY && !ctx && pending == 0);
        most = ~0ull;
    }
    if (create(&ctx, 0, 3000, 8192) != MAKO_OK) {
        printf("no context\n");
        return 1;
    }
    alignas(16) static char memory[64]; // (nothing is read there: no kernel runs)
    int32_t* const ints = reinterpret_cast<int32_t*>(memory);

    mako_cut_desc cut;
    memset(&cut, 0, sizeof cut);
    cut.logits = cut.params = reinterpret_cast<mako_sampling_params*>(memory);
    cut.out_cuts = reinterpret_cast<mako_row_cut*>(memory);
    cut.n_rows = 4;
    cut.n_vocab = 1000;
    cut.logits_stride = cut.probs_stride = 8192;
    mako_cut_desc wide = cut, dense;
    wide.n_vocab = 8192;
    dense = wide;
    dense.out_probs = reinterpret_cast<float*>(memory);

    mako_verify_desc verify;
    memset(&verify, 0, sizeof verify);
    verify.n_requests = 4;
    verify.n_vocab = 1000;
    verify.target = memory;
    verify.target_stride = 1000;
    verify.u = reinterpret_cast<float*>(memory);
    verify.out_tokens = verify.out_accepted = ints;

    mako_blocks_desc blocks;
    memset(&blocks, 0, sizeof blocks);
    blocks.n_requests = 4;
    blocks.block_size = 16;
    blocks.seq_len = blocks.new_len = ints;
    blocks.block_table = blocks.free_blocks = blocks.out_start = blocks.out_status = ints;
    blocks.n_blocks = blocks.n_free = ints;
    blocks.out_n_blocks = blocks.out_n_free = ints; // (in place)
    blocks.table_stride = blocks.max_blocks = 8;
    blocks.free_capacity = 8;
    blocks.max_tokens = 16;
    blocks.out_slots = reinterpret_cast<int64_t*>(memory);
    mako_blocks_desc many_tokens = blocks, many_requests = blocks;
    many_tokens.max_tokens = 5000;
    many_requests.n_requests = 3000;

    const auto each = [&](auto f) {
        f("cut", 2, [&] { return cut_rows(ctx, &cut, nullptr); });
        f("cut with lists", 4, [&] { return cut_rows(ctx, &wide, nullptr); });
        f("cut with probabilities", 5, [&] { return cut_rows(ctx, &dense, nullptr); });
        f("verify", 2, [&] { return verify_drafts(ctx, &verify, nullptr); });
        f("blocks", 1, [&] { return assign_blocks(ctx, &blocks, nullptr); });
        f("blocks of many tokens", 2, [&] { return assign_blocks(ctx, &many_tokens, nullptr); });
        f("blocks of many requests", 2, [&] { return assign_blocks(ctx, &many_requests, nullptr); });
    };
    each([&](const char* name, int n, auto call) {
        launches = 0;
        expect(name, "fails where nothing does", call() == MAKO_OK && launches == n);
        // an error of some earlier call, which nobody has looked at yet, is not this call's
        launches = 0;
        pending = kNotReady;
        expect(name, "takes an earlier error for its own", call() == MAKO_OK && launches == n);
        pending = 0;
        // a launch that fails is the last, and the call's alone
        for (failing = 1; failing <= n; ++failing) {
            launches = 0;
            expect(name, "does not report a failed launch", call() == MAKO_ERR_HIP && strstr(last_error(ctx), "could not be launched"));
            expect(name, "goes on behind a failed launch", launches == failing);
            expect(name, "leaves its error to the next call", pending == 0);
            pending = 0;
        }
        failing = 0;
    });
    destroy(ctx);
    if (!failures)
        printf("ok\n");
    return failures ? 1 : 0;
}
