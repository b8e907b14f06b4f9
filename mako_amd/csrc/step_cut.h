// What the kernels that cut rows share: what a row's parameters ask of the pass over it.
#pragma once

#include "step_common.h"
#include "step_launch.h"

namespace mako {
namespace step {

// Rows of no more logits than this are held whole where they are cut, and have no lists: 64 rows of 6144 cut to a top_p take 19 us, of
// 6145 with lists 36, to a top_k of 50 14 and 16.  (The more are held, the fewer workgroups a CU has: 49 of 160 KB of LDS here.)
constexpr uint32_t kWholeRow = 6144;

// Largest top_k that is looked for in the chunks' lists, of a row and of a chunk's share of it.  (64 rows of 129280, 64 chunks: top_k
// 2000 takes 27 us, and 45 with its weights summed up and a pass around its cut; 4000, by that way, 53.)
constexpr uint32_t kListTopK = 2500, kListShare = 32;

struct RowKind {
    bool greedy, cut; // cut: something may be cut off it, and the chunks' first tokens are wanted
    bool min_p, top_p;
    bool listed;      // the first top_k tokens are to be expected in the lists
    bool sums;        // the weights' sums are wanted (not of those: they are added up alone)
    uint32_t top_k;
    double scale;     // of weights: log2(e) / T

    __device__ __forceinline__ RowKind(const mako_sampling_params& p, uint32_t n_vocab)
    {
        greedy = !(p.temperature > 0.0f);
        min_p = !greedy && p.min_p > 0.0f;
        top_p = !greedy && p.top_p < 1.0f;
        top_k = greedy ? 0u : p.top_k;
        cut = min_p || top_p || top_k;
        listed = top_k && top_k < n_vocab && top_k <= (n_vocab <= kWholeRow ? kListTopK : min(kListTopK, kListShare * chunks_of(n_vocab)));
        sums = !greedy && !listed;
        scale = weight_scale(p.temperature);
    }
    // Lanes of a chunk's 64 whose largest logit should be in its list.  What a top_k takes of a chunk if chance spreads its tokens, the
    // mean and some four deviations and three, and a fifth of that again for how chance spreads them over the lanes: t tokens leave
    // 64 exp(-t / 64) lanes without one (t is 71 at most, well below the 128 that there is room for).  Without such a top_k,
    // enough for a narrow nucleus (64 rows of 129280, N(0, 4^2) and N(0, 5^2): 45 and 23 us; with 20 lanes 44 and 25), and more for a
    // min_p, which has no other way (0.02 of N(0, 3^2): 27.5 us; 12 lanes 61, 40 lanes 30).
    __device__ __forceinline__ uint32_t list_length(uint32_t chunks) const
    {
        if (!listed)
            return min_p ? 24u : 10u;
        const float mean = (float)top_k / (float)chunks, t = 1.2f * (mean + 4.2f * sqrtf(mean) + 3.0f);
        return (uint32_t)(65.0f - 64.0f * __builtin_amdgcn_exp2f(-(1.4426950f / 64.0f) * t));
    }
};

} // namespace step
} // namespace mako
