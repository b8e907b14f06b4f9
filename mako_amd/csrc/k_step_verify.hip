// Verification of drafted tokens (mako_step_verify_drafts).
//
//   left_kernel  a workgroup for every part of 4096 tokens of every request: where the request stops accepting, and what
//                the slice has left there to draw from
//   draw_kernel  a workgroup for every request: the slice that the uniform falls into, and the token in it
#include "step_common.h"
#include "step_launch.h"

namespace mako {
namespace step {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr uint32_t kRun = 8, kRuns = kPart / kThreads / kRun; // a thread has runs of 8 tokens: of either row, whatever its type

// A row of weights: logits under their cut, or probabilities.
template <class E>
struct Row {
    const typename E::raw* x;
    const uint32_t* mask;
    uint32_t n;
    bool probs;
    float cut;
    int32_t cut_token;
    double max, scale, share;

    __device__ __forceinline__ Row(const void* base, int64_t stride, const uint32_t* masks, int64_t mask_stride, const mako_row_cut* cuts, uint32_t n_vocab, uint64_t row)
        : x(static_cast<const typename E::raw*>(base) + (int64_t)row * stride), mask(cuts && masks ? masks + (int64_t)row * mask_stride : nullptr), n(n_vocab),
          probs(!cuts), cut(0.0f), cut_token(-1), max(0.0), scale(0.0), share(0.0)
    {
        if (cuts) {
            const mako_row_cut c = cuts[row];
            cut = c.cut_logit;
            cut_token = c.cut_token;
            max = (double)c.max_logit;
            scale = weight_scale(c.temperature);
            share = c.total > 0.0 ? 1.0 / c.total : 0.0;
        }
    }
    __device__ __forceinline__ double prob(uint32_t i, float v) const // (v: as token_logit() gives it, or a probability)
    {
        if (probs)
            return v > 0.0f && v <= kFltMax ? (double)v : 0.0;
        const bool kept = v > cut || (v == cut && (int32_t)i <= cut_token);
        return kept ? weight(v, max, scale) * share : 0.0;
    }
    __device__ __forceinline__ double one(uint32_t i) const
    {
        if (i >= n)
            return 0.0;
        const float v = E::of(x[i], 0);
        return prob(i, probs ? v : token_logit(v, !mask || (mask[i >> 5] >> (i & 31u) & 1u)));
    }
    // kRun probabilities from token i on; 0 behind the row's end
    __device__ __forceinline__ void run(uint32_t i, double* p) const
    {
        float v[kRun];
#pragma unroll
        for (uint32_t h = 0; h < kRun; h += E::kVec) {
            if (probs)
                load_vec<E>(x, i + h, n, v + h);
            else
                load_tokens<E>(x, mask, i + h, n, v + h);
        }
#pragma unroll
        for (uint32_t k = 0; k < kRun; ++k)
            p[k] = prob(i + k, v[k]);
    }
};

// What there is to draw from behind the last accepted draft: p, p without a token, or max(0, p - q).
template <class E, class Q>
struct Left {
    Row<E> p;
    Row<Q> q;
    bool minus_q;
    uint32_t without; // kNoToken: none

    __device__ __forceinline__ void run(uint32_t i, double* r) const
    {
        p.run(i, r);
        if (minus_q) {
            double s[kRun];
            q.run(i, s);
#pragma unroll
            for (uint32_t k = 0; k < kRun; ++k)
                r[k] = fmax(r[k] - s[k], 0.0);
        }
#pragma unroll
        for (uint32_t k = 0; k < kRun; ++k)
            if (i + k == without)
                r[k] = 0.0;
    }
    __device__ __forceinline__ void give_up()
    {
        minus_q = false;
        without = kNoToken;
    }
    // (16 tokens of a slice of 4096 to a thread; the sum of the thread's own)
    __device__ __forceinline__ double slice(uint32_t s, double* r) const
    {
        double sum = 0.0;
#pragma unroll
        for (uint32_t j = 0; j < kRuns; ++j)
            run(s * kPart + (j * kThreads + threadIdx.x) * kRun, r + j * kRun);
#pragma unroll
        for (int k = 0; k < 16; ++k)
            sum += r[k];
        return sum;
    }
};

__device__ __forceinline__ uint32_t drafts_of(const mako_verify_desc& d, uint32_t b, bool& there)
{
    const int32_t n = d.n_drafts ? d.n_drafts[b] : (int32_t)d.max_drafts;
    there = n >= 0;
    return there ? min((uint32_t)n, d.max_drafts) : 0u;
}

template <class E>
__device__ __forceinline__ Row<E> target_row(const mako_verify_desc& d, uint64_t row)
{
    return Row<E>(d.target, d.target_stride, d.target_mask, d.target_mask_stride, d.target_cuts, d.n_vocab, row);
}
template <class E>
__device__ __forceinline__ Row<E> draft_row(const mako_verify_desc& d, uint64_t row)
{
    return Row<E>(d.draft, d.draft_stride, d.draft_mask, d.draft_mask_stride, d.draft_cuts, d.n_vocab, row);
}

// Drafts that request b accepts: a lane of the wave for each.
template <class E, class Q>
__device__ __forceinline__ uint32_t accepted_drafts(const mako_verify_desc& d, uint32_t b, uint32_t drafts)
{
    const uint32_t j = (uint32_t)lane();
    bool stop = j >= drafts;
    if (!stop) {
        const uint32_t token = (uint32_t)d.draft_tokens[(uint64_t)b * d.max_drafts + j];
        const double p = target_row<E>(d, (uint64_t)b * (d.max_drafts + 1) + j).one(token);
        const double q = d.draft ? draft_row<Q>(d, (uint64_t)b * d.max_drafts + j).one(token) : 1.0;
        stop = !((double)d.u[(uint64_t)b * (d.max_drafts + 1) + j] * q < p);
    }
    const unsigned long long stops = __ballot(stop);
    return min(stops ? (uint32_t)__builtin_ctzll(stops) : 64u, drafts);
}

template <class E, class Q>
__device__ __forceinline__ Left<E, Q> left_of(const mako_verify_desc& d, uint32_t b, uint32_t accepted, uint32_t drafts)
{
    const bool rejected = accepted < drafts;
    const bool minus_q = rejected && d.draft;
    Left<E, Q> left = {target_row<E>(d, (uint64_t)b * (d.max_drafts + 1) + accepted),
                      minus_q ? draft_row<Q>(d, (uint64_t)b * d.max_drafts + accepted) : Row<Q>(nullptr, 0, nullptr, 0, nullptr, d.n_vocab, 0), minus_q, kNoToken};
    if (rejected && !d.draft)
        left.without = (uint32_t)d.draft_tokens[(uint64_t)b * d.max_drafts + accepted];
    return left;
}

template <class E, class Q>
__global__ void __launch_bounds__(kThreads) left_kernel(mako_verify_desc d, Scratch sc)
{
    __shared__ Share<kWaves> share;
    const uint32_t b = blockIdx.y;
    bool there;
    const uint32_t drafts = drafts_of(d, b, there);
    if (!there)
        return;
    const uint32_t accepted = accepted_drafts<E, Q>(d, b, drafts);
    const Left<E, Q> left = left_of<E, Q>(d, b, accepted, drafts);
    double r[16];
    const double sum = all_sum<kWaves>(left.slice(blockIdx.x, r), share);
    if (threadIdx.x == 0) {
        sc.parts[(uint64_t)b * sc.parts_cap + blockIdx.x] = sum;
        if (blockIdx.x == 0)
            sc.stop[b] = accepted;
    }
}

template <class E, class Q>
__global__ void __launch_bounds__(kThreads) draw_kernel(mako_verify_desc d, Scratch sc)
{
    __shared__ Share<kWaves> share;
    __shared__ double found_before;
    const uint32_t b = blockIdx.x, places = d.max_drafts + 1;
    bool there;
    const uint32_t drafts = drafts_of(d, b, there);
    if (!there)
        return;
    const uint32_t accepted = sc.stop[b];
    Left<E, Q> left = left_of<E, Q>(d, b, accepted, drafts);
    const uint32_t slices = (d.n_vocab + kPart - 1) / kPart;
    double* parts = sc.parts + (uint64_t)b * sc.parts_cap;
    double r[16];
    // the slices: one to a thread (no more than 256 of them)
    double part = threadIdx.x < slices ? parts[threadIdx.x] : 0.0, total;
    double before = sum_before<kWaves>(part, total, share);
    if (!(total > 0.0)) {
        // nothing is left: from p itself
        left.give_up();
        for (uint32_t s = 0; s < slices; ++s) {
            const double sum = all_sum<kWaves>(left.slice(s, r), share);
            if (threadIdx.x == s)
                part = sum;
        }
        before = sum_before<kWaves>(part, total, share);
    }
    uint32_t token = kNoToken;
    if (total > 0.0) {
        const double goal = (double)d.u[(uint64_t)b * places + d.max_drafts] * total;
        // the first slice, then the first token, with which the running sum exceeds the goal; should rounding leave none, the
        // last that has a weight
        const uint32_t first = all_min<kWaves>(part > 0.0 && before + part > goal ? threadIdx.x : kNoToken, share);
        const uint32_t last = ~all_min<kWaves>(part > 0.0 ? ~threadIdx.x : kNoToken, share);
        const uint32_t at = first != kNoToken ? first : last;
        if (threadIdx.x == at)
            found_before = before;
        __syncthreads();
        left.slice(at, r);
        double run = found_before;
        uint32_t hit = kNoToken, weighty = 0; // (weighty: a token + 1)
#pragma unroll
        for (uint32_t j = 0; j < kRuns; ++j) {
            const uint32_t i = at * kPart + (j * kThreads + threadIdx.x) * kRun;
            double mine = 0.0, all;
#pragma unroll
            for (uint32_t k = 0; k < kRun; ++k)
                mine += r[j * kRun + k];
            double here = run + sum_before<kWaves>(mine, all, share);
#pragma unroll
            for (uint32_t k = 0; k < kRun; ++k) {
                const double w = r[j * kRun + k];
                here += w;
                if (w > 0.0) {
                    weighty = i + k + 1u;
                    if (here > goal && hit == kNoToken)
                        hit = i + k;
                }
            }
            run += all;
        }
        hit = all_min<kWaves>(hit, share);
        weighty = ~all_min<kWaves>(~weighty, share);
        token = hit != kNoToken ? hit : weighty - 1u;
    }
    for (uint32_t j = threadIdx.x; j < places; j += kThreads)
        d.out_tokens[(uint64_t)b * places + j] = j < accepted ? d.draft_tokens[(uint64_t)b * d.max_drafts + j] : (j == accepted ? (int32_t)token : -1);
    if (threadIdx.x == 0) {
        d.out_accepted[b] = (int32_t)accepted;
        if (d.seq_len)
            d.out_seq_len[b] = d.seq_len[b] + (int32_t)accepted + (token != kNoToken);
    }
}

template <class E, class Q>
void verify(hipStream_t st, const mako_verify_desc& d, const Scratch& sc)
{
    hipLaunchKernelGGL((left_kernel<E, Q>), dim3((d.n_vocab + kPart - 1) / kPart, d.n_requests), dim3(kThreads), 0, st, d, sc);
    hipLaunchKernelGGL((draw_kernel<E, Q>), dim3(d.n_requests), dim3(kThreads), 0, st, d, sc);
}
template <class E>
void verify(hipStream_t st, const mako_verify_desc& d, const Scratch& sc)
{
    const uint32_t q = d.draft ? d.draft_type : d.target_type;
    q == MAKO_LOGITS_F32 ? verify<E, F32>(st, d, sc) : (q == MAKO_LOGITS_BF16 ? verify<E, BF16>(st, d, sc) : verify<E, F16>(st, d, sc));
}

} // namespace

void launch_verify(hipStream_t st, const mako_verify_desc& d, const Scratch& sc)
{
    d.target_type == MAKO_LOGITS_F32 ? verify<F32>(st, d, sc) : (d.target_type == MAKO_LOGITS_BF16 ? verify<BF16>(st, d, sc) : verify<F16>(st, d, sc));
}

} // namespace step
} // namespace mako
