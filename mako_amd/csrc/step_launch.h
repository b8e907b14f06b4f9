// The launchers of the step's kernels (one translation unit per operator) and the scratch memory that they are given.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/mako_step.h"

namespace mako {
namespace step {

// A row is read in chunks of 2048 logits, a wave each.
constexpr uint32_t kChunk = 2048;
constexpr uint32_t kChunkList = 128; // a chunk's first tokens that are written out, at most
constexpr uint32_t kLookList = 512;  // ... and those around the row's cut

// (what the second pass over a row, around its cut, finds in a chunk takes the same place: `sum` of the tokens that are weighed,
// `count` of those above, `n_list` in the list)
struct ChunkRec {
    double sum;      // of the weights, relative to the chunk's own largest logit (rows that need their total)
    float max;       // -inf: no token
    float listed;    // all tokens of this logit and above are in the list; +inf: none
    uint32_t count;  // tokens
    uint32_t n_list;
    uint32_t first;  // the first token of the largest logit (rows without lists)
    float low;       // the smallest logit (rows with a min_p)
};

// A row whose cut lies further down than the chunks' lists: what the second pass looks for.
struct RowPlan {
    double mass, total; // the cut is behind the first tokens that weigh `mass`, of all that weigh `total` (if that is known),
    uint32_t rank;      // or, if not 0, behind the first `rank`
    uint32_t row, tokens; // which row, and how many tokens it has
    float max;          // its largest logit
    double scale;       // log2(e) / T
    float low, high;    // the tokens from `low` up to `high` are listed,
    uint32_t from_above; // those above are weighed, or those below
    float top_p;        // of what the first `rank` weigh; 1: none
    uint32_t sums;      // `total` is known
    uint32_t look;       // 0: there is no guess where it lies
};

// Where a request stops accepting, and what its rows there need: a row's cut with its divisions made.
struct StopRow {
    double max, scale, share; // a kept token's probability is 2^((logit - max) scale) share
    float cut;
    int32_t cut_token;
};
struct Stop {
    StopRow target, draft;
    uint32_t accepted, rejected; // drafts it accepts, and whether there is one that it does not
    uint32_t without, reserved;  // a token that is not drawn; 0xffffffff: none
};

struct Scratch {
    ChunkRec* chunks;     // [rows][chunks_cap]
    uint64_t* lists;      // [rows][chunks_cap][kChunkList]: a token's number, and its logit above that (null, like looks, where no row
                          // is longer than what is held whole)
    uint64_t* looks;      // [rows][chunks_cap][kLookList]: by plan (and the chunks too, then)
    uint32_t chunks_cap;  // of a row
    RowPlan* plans;       // [rows]: of those that have one, in no order
    uint32_t* wide;       // [1]: how many do
    double* parts;        // [rows][parts_cap]: what is left to draw from in each part of the row where a request stops
    uint32_t parts_cap;
    Stop* stops;          // [rows]
    uint32_t* released;   // [rows + 1] blocks given back by the requests before
    uint32_t* taken;      // [rows + 1] blocks taken by the requests before
    uint32_t* held;       // [rows] blocks a request keeps before it takes any
    uint32_t* start;      // [rows + 1] new tokens of the requests before
    uint32_t* free_state; // [2] blocks on the free list before the call, and after the releases
};

__host__ __device__ inline uint32_t chunks_of(uint32_t n_vocab)
{
    return (n_vocab + kChunk - 1) / kChunk;
}

// A kernel's launch, with its own status.
template <class T>
struct Given {
    using type = T;
};
template <class... P>
hipError_t launch(void (*kernel)(P...), dim3 grid, uint32_t threads, size_t lds, hipStream_t st, typename Given<P>::type... args)
{
    void* at[] = {&args...};
    return hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, dim3(threads), at, lds, st);
}

// (of more than one launch, the first that fails is the last: the kernels behind it would work on what it did not write)
hipError_t launch_scan(hipStream_t st, const mako_cut_desc& d, const Scratch& sc);
hipError_t launch_look(hipStream_t st, const mako_cut_desc& d, const Scratch& sc);
hipError_t launch_cut(hipStream_t st, const mako_cut_desc& d, const Scratch& sc);
hipError_t launch_probs(hipStream_t st, const mako_cut_desc& d);
hipError_t launch_verify(hipStream_t st, const mako_verify_desc& d, const Scratch& sc);
hipError_t launch_blocks(hipStream_t st, const mako_blocks_desc& d, const Scratch& sc);
hipError_t init_cut();

} // namespace step
} // namespace mako
