// The launchers of the step's kernels (one translation unit per operator) and the scratch memory that they are given.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/mako_step.h"

namespace mako {
namespace step {

// What a wave finds in its chunk of a row.
struct ChunkRec {
    double sum;     // of the weights, relative to the chunk's own largest logit
    float max;      // -inf: no token
    uint32_t count; // of tokens
};

// Of a batch of requests: where a request stopped accepting, and what is left to draw from in each slice of that row.
struct Scratch {
    ChunkRec* chunks;     // [rows][chunks_cap]
    uint32_t chunks_cap;  // of a row
    double* parts;        // [rows][slices_cap]
    uint32_t slices_cap;
    uint32_t* stop;       // [rows]
    uint32_t* released;   // [rows + 1] blocks given back by the requests before
    uint32_t* taken;      // [rows + 1] blocks taken by the requests before
    uint32_t* held;       // [rows] blocks a request keeps before it takes any
    uint32_t* free_state; // [2] blocks on the free list before the call, and after the releases
};

void launch_cut(hipStream_t st, const mako_cut_desc& d, const Scratch& sc);
void launch_probs(hipStream_t st, const mako_cut_desc& d);
void launch_verify(hipStream_t st, const mako_verify_desc& d, const Scratch& sc);
void launch_blocks(hipStream_t st, const mako_blocks_desc& d, const Scratch& sc);
hipError_t init_cut();

} // namespace step
} // namespace mako
