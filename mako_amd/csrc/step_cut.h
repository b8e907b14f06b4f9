// What the kernels that cut rows share: what a row's parameters ask of the pass over it.
#pragma once

#include "step_common.h"
#include "step_launch.h"

namespace mako {
namespace step {

// Largest top_k that is looked for in the chunks' lists.
constexpr uint32_t kListTopK = 1024;

// Rows of no more logits than this are held whole where they are cut, and have no lists.
constexpr uint32_t kWholeRow = 6144;

struct RowKind {
    bool greedy, cut; // cut: something may be cut off it, and the chunks' first tokens are wanted
    bool min_p, top_p;
    bool sums;        // the weights' sums are wanted (not where a top_k leaves few tokens: these are added up alone)
    uint32_t top_k;
    double scale;     // of weights: log2(e) / T

    __device__ __forceinline__ explicit RowKind(const mako_sampling_params& p)
    {
        greedy = !(p.temperature > 0.0f);
        min_p = !greedy && p.min_p > 0.0f;
        top_p = !greedy && p.top_p < 1.0f;
        top_k = greedy ? 0u : p.top_k;
        cut = min_p || top_p || top_k;
        sums = !greedy && (top_k == 0 || top_k > kListTopK);
        scale = weight_scale(p.temperature);
    }
    // Lanes of a chunk's 64 whose largest logit should be in its list: what a top_k takes of a chunk if chance spreads its tokens
    // (the mean, and three and a half deviations; at most 52, whose logits and those above are some 105 tokens of 2048); without a
    // top_k, enough for a narrow nucleus, and more for a min_p, which has no other way.
    __device__ __forceinline__ uint32_t list_length(uint32_t chunks) const
    {
        const float mean = (float)min(top_k, kListTopK) / (float)chunks;
        return top_k && top_k <= kListTopK ? min((uint32_t)(mean + 3.5f * sqrtf(mean)) + 4u, 52u) : (min_p ? 24u : 10u);
    }
};

} // namespace step
} // namespace mako
