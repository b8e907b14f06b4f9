// Verification of drafted tokens (mako_step_verify_drafts).
//
//   left_kernel  a workgroup for every part of 1024 tokens of every request, or for several: where the request stops accepting,
//                which each of them finds out for itself, and what its parts have left there to draw from
//   draw_kernel  a workgroup for every request: the part that the uniform falls into, and the token in it
//
// Of a request's rows only one is read whole, the one behind the last accepted draft, and of the drafter's the one beside it: which
// these are follows from one logit of each row, which every workgroup looks up for itself (a launch of its own would cost more).
// What is left, max(0, p - q), is needed as a sum before a token can be drawn by it: the parts' sums first, then one part again.
// 64 requests over 129280 bf16 logits of each kind (33 MB) take 14.6 and 5.0 us, one over 151552 fp32 logits 5.6 and 4.4, 32 with
// looked-up drafts under masks 7.6 and 5.1, 256 over 32000 probabilities (66 MB) 12.6 and 4.6: large ones are bound by
// memory and the weights' arithmetic (two weights of 20 instructions a token), small ones by five trips to memory in a row, draw_kernel
// always.
#include "step_common.h"
#include "step_launch.h"

namespace mako {
namespace step {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr uint32_t kMostParts = 32; // of a workgroup
static_assert(kPart == 4 * kThreads, "four tokens to a thread");

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

    __device__ __forceinline__ Row(const void* base, int64_t stride, const uint32_t* masks, int64_t mask_stride, bool cuts, const StopRow& c, uint32_t n_vocab, uint64_t row)
        : x(static_cast<const typename E::raw*>(base) + (int64_t)row * stride), mask(cuts && masks ? masks + (int64_t)row * mask_stride : nullptr), n(n_vocab),
          probs(!cuts), cut(c.cut), cut_token(c.cut_token), max(c.max), scale(c.scale), share(c.share)
    {
    }
    // Whether a logit as it is in memory can be one of a kept token; probabilities: whether it is one.
    __device__ __forceinline__ bool may_keep(float v) const { return probs ? v > 0.0f : v >= cut; }
    // (v: as token_logit() gives it, or a probability)
    __device__ __forceinline__ bool kept(uint32_t i, float v) const
    {
        return probs ? v > 0.0f && v <= kFltMax : v > cut || (v == cut && (int32_t)i <= cut_token);
    }
    __device__ __forceinline__ double one(uint32_t i, float v, uint32_t bits) const
    {
        if (!probs)
            v = token_logit(v, bits >> (i & 31u) & 1u);
        if (i >= n || !kept(i, v))
            return 0.0;
        return probs ? (double)v : weight(v, max, scale) * share;
    }
    // four logits or probabilities from token i on, as they are in memory; whole: none is behind the row's end
    __device__ __forceinline__ void load(uint32_t i, bool whole, float* v) const
    {
        if (whole)
            load_whole_four<E>(x, i, v);
        else
            load_four<E>(x, i, n, v);
    }
    // and the probabilities that these are
    __device__ __forceinline__ void four(uint32_t i, const float* v, double* out) const
    {
        if (probs) {
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k)
                out[k] = kept(i + k, v[k]) ? (double)v[k] : 0.0;
            return;
        }
        uint32_t bits = 0xffffffffu;
        if (mask) // (the four bits lie in one word)
            bits = i < n ? mask[i >> 5] >> (i & 31u) : 0u;
        float x4[4];
        double t[4];
#pragma unroll
        for (uint32_t k = 0; k < 4u; ++k) {
            x4[k] = token_logit(v[k], (bits >> k) & 1u);
            t[k] = ((double)x4[k] - max) * scale;
        }
        exp2_down<4>(t, out);
#pragma unroll
        for (uint32_t k = 0; k < 4u; ++k)
            out[k] = kept(i + k, x4[k]) ? out[k] * share : 0.0;
    }
};

// What there is to draw from behind the last accepted draft: p, p without a token, or max(0, p - q).
template <class E, class Q>
struct Left {
    Row<E> p;
    Row<Q> q;
    bool minus_q;
    uint32_t without; // kNoToken: none

    __device__ __forceinline__ void give_up()
    {
        minus_q = false;
        without = kNoToken;
    }
    // p's tokens of a part, four to a thread; whether any of the wave's may have something left; and q's
    __device__ __forceinline__ void load_p(uint32_t at, float* v) const { p.load(at * kPart + threadIdx.x * 4u, (at + 1u) * kPart <= p.n, v); }
    __device__ __forceinline__ bool any(const float* v) const
    {
        return __ballot(p.may_keep(v[0]) || p.may_keep(v[1]) || p.may_keep(v[2]) || p.may_keep(v[3])) != 0;
    }
    __device__ __forceinline__ void load_q(uint32_t at, float* w) const
    {
        if (minus_q)
            q.load(at * kPart + threadIdx.x * 4u, (at + 1u) * kPart <= p.n, w);
    }
    // and what they have left
    __device__ __forceinline__ void four(uint32_t at, const float* v, const float* w, double* r) const
    {
        const uint32_t i = at * kPart + threadIdx.x * 4u;
        p.four(i, v, r);
        if (minus_q) {
            double s[4];
            q.four(i, w, s);
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k)
                r[k] = fmax(r[k] - s[k], 0.0);
        }
#pragma unroll
        for (uint32_t k = 0; k < 4u; ++k)
            if (i + k == without)
                r[k] = 0.0;
    }
    __device__ __forceinline__ void part(uint32_t at, double* r) const
    {
        float v[4], w[4];
        load_p(at, v);
        r[0] = r[1] = r[2] = r[3] = 0.0;
        if (any(v)) {
            load_q(at, w);
            four(at, v, w, r);
        }
    }
};

template <class E>
__device__ __forceinline__ Row<E> target_row(const mako_verify_desc& d, const StopRow& c, uint64_t row)
{
    return Row<E>(d.target, d.target_stride, d.target_mask, d.target_mask_stride, d.target_cuts != nullptr, c, d.n_vocab, row);
}
template <class E>
__device__ __forceinline__ Row<E> draft_row(const mako_verify_desc& d, const StopRow& c, uint64_t row)
{
    return Row<E>(d.draft, d.draft_stride, d.draft_mask, d.draft_mask_stride, d.draft_cuts != nullptr, c, d.n_vocab, row);
}

__device__ __forceinline__ StopRow stop_row(const mako_row_cut& c)
{
    return {(double)c.max_logit, weight_scale(c.temperature), c.total > 0.0 ? 1.0 / c.total : 0.0, c.cut_logit, c.cut_token};
}
template <class T>
union Words {
    T value;
    int words[sizeof(T) / 4];
};
template <class T>
__device__ __forceinline__ T of_lane(const T& v, uint32_t from)
{
    Words<T> u;
    u.value = v;
#pragma unroll
    for (uint32_t k = 0; k < sizeof(T) / 4u; ++k)
        u.words[k] = __builtin_amdgcn_readlane(u.words[k], (int)from);
    return u.value;
}

// Where request b stops: a lane of the wave for each draft.  Everything but the drafts' own logits is asked for at once.
template <class E, class Q>
__device__ __forceinline__ Stop find_stop(const mako_verify_desc& d, uint32_t b, int32_t n_drafts)
{
    const uint32_t k = d.max_drafts, j = (uint32_t)lane();
    const uint64_t p_row = (uint64_t)b * (k + 1), q_row = (uint64_t)b * k;
    mako_row_cut p_cut = {}, q_cut = {};
    uint32_t token = kNoToken;
    float u = 1.0f;
    if (j <= k && d.target_cuts)
        p_cut = d.target_cuts[p_row + j];
    if (j < k) {
        token = (uint32_t)d.draft_tokens[q_row + j];
        u = d.u[p_row + j];
        if (d.draft && d.draft_cuts)
            q_cut = d.draft_cuts[q_row + j];
    }
    StopRow p_stop = stop_row(p_cut);
    const StopRow q_stop = stop_row(q_cut);
    const Row<E> p = target_row<E>(d, p_stop, p_row + j);
    const Row<Q> q = draft_row<Q>(d, q_stop, q_row + j);
    float p_logit = 0.0f, q_logit = 0.0f;
    uint32_t p_bits = ~0u, q_bits = ~0u;
    if (token < d.n_vocab) {
        p_logit = E::of(p.x[token], 0);
        if (p.mask)
            p_bits = p.mask[token >> 5];
        if (d.draft) {
            q_logit = Q::of(q.x[token], 0);
            if (q.mask)
                q_bits = q.mask[token >> 5];
        }
    }
    const uint32_t drafts = min((uint32_t)max(n_drafts, 0), k);
    const bool stops = j >= drafts || !((double)u * (d.draft ? q.one(token, q_logit, q_bits) : 1.0) < p.one(token, p_logit, p_bits));
    const unsigned long long all = __ballot(stops);
    Stop stop;
    stop.accepted = all ? (uint32_t)__builtin_ctzll(all) : 64u;
    stop.rejected = stop.accepted < drafts;
    const uint32_t at = min(stop.accepted, 63u);
    stop.target = of_lane(p_stop, at);
    stop.draft = of_lane(q_stop, at);
    if (stop.accepted == 64u && d.target_cuts) // (as many drafts as lanes, and all are accepted)
        stop.target = stop_row(d.target_cuts[p_row + 64u]);
    stop.without = stop.rejected && !d.draft ? (uint32_t)__builtin_amdgcn_readlane((int)token, (int)at) : kNoToken;
    stop.reserved = 0;
    return stop;
}

template <class E, class Q>
__device__ __forceinline__ Left<E, Q> left_of(const mako_verify_desc& d, uint32_t b, const Stop& stop)
{
    return {target_row<E>(d, stop.target, (uint64_t)b * (d.max_drafts + 1) + stop.accepted), draft_row<Q>(d, stop.draft, (uint64_t)b * d.max_drafts + stop.accepted),
            stop.rejected && d.draft, stop.without};
}

template <class E, class Q>
__global__ void __launch_bounds__(kThreads, 8) left_kernel(mako_verify_desc d, Scratch sc, uint32_t each)
{
    __shared__ double sums[kMostParts][kWaves];
    __shared__ Words<Stop> shared;
    const uint32_t b = blockIdx.y, parts = (d.n_vocab + kPart - 1) / kPart, first = blockIdx.x * each, n = min(each, parts - first);
    const int32_t n_drafts = d.n_drafts ? d.n_drafts[b] : (int32_t)d.max_drafts;
    // (one wave finds the place: by all of them that alone took as long as the rest)
    if (wave() == 0) {
        const Stop found = find_stop<E, Q>(d, b, n_drafts);
        if (threadIdx.x == 0) {
            shared.value = found;
            if (blockIdx.x == 0)
                sc.stops[b] = found;
        }
    }
    __syncthreads();
    if (n_drafts < 0)
        return;
    Words<Stop> known;
#pragma unroll
    for (uint32_t k = 0; k < sizeof(Stop) / 4u; ++k)
        known.words[k] = __builtin_amdgcn_readfirstlane(shared.words[k]);
    const Left<E, Q> left = left_of<E, Q>(d, b, known.value);
    // (p's tokens are on their way two parts ahead, q's one, and only where a wave's 256 tokens of p have something left: in a row cut
    // to a narrow nucleus most have not)
    float v[4], w[4], next_v[4];
    left.load_p(first, v);
    if (n > 1u)
        left.load_p(first + 1u, next_v);
    bool here = left.any(v);
    if (here)
        left.load_q(first, w);
#pragma unroll 1
    for (uint32_t j = 0; j < n; ++j) {
        float next_w[4], after_v[4];
        const bool next = j + 1u < n && left.any(next_v);
        if (next)
            left.load_q(first + j + 1u, next_w);
        if (j + 2u < n)
            left.load_p(first + j + 2u, after_v);
        double sum = 0.0;
        if (here) {
            double r[4];
            left.four(first + j, v, w, r);
            sum = __ockl_wfred_add_f64(r[0] + r[1] + r[2] + r[3]);
        }
        if (lane() == 0)
            sums[j][wave()] = sum;
        here = next;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v[k] = next_v[k];
            w[k] = next_w[k];
            next_v[k] = after_v[k];
        }
    }
    __syncthreads();
    if (threadIdx.x < n) {
        double sum = 0.0;
        for (int k = 0; k < kWaves; ++k)
            sum += sums[threadIdx.x][k];
        sc.parts[(uint64_t)b * sc.parts_cap + first + threadIdx.x] = sum;
    }
}

template <class E, class Q>
__global__ void __launch_bounds__(kThreads) draw_kernel(mako_verify_desc d, Scratch sc)
{
    __shared__ Share<kWaves> share;
    __shared__ double found_before;
    const uint32_t b = blockIdx.x, places = d.max_drafts + 1, parts = (d.n_vocab + kPart - 1) / kPart;
    const int32_t n_drafts = d.n_drafts ? d.n_drafts[b] : 0;
    const Stop stop = sc.stops[b]; // (of a request that is not there: not looked at)
    // the parts: four to a thread (no more than 1024 of them)
    static_assert(MAKO_STEP_MAX_VOCAB / kPart <= 4 * kThreads, "parts of a row");
    double part[4], r[4], total;
#pragma unroll
    for (uint32_t k = 0; k < 4u; ++k)
        part[k] = threadIdx.x * 4u + k < parts ? sc.parts[(uint64_t)b * sc.parts_cap + threadIdx.x * 4u + k] : 0.0;
    const float u = d.u[(uint64_t)b * places + d.max_drafts];
    int32_t draft = -1;
    if (threadIdx.x < d.max_drafts)
        draft = d.draft_tokens[(uint64_t)b * d.max_drafts + threadIdx.x];
    const int32_t length = d.seq_len ? d.seq_len[b] : 0;
    if (n_drafts < 0)
        return;
    Left<E, Q> left = left_of<E, Q>(d, b, stop);
    double before = sum_before<kWaves>(part[0] + part[1] + part[2] + part[3], total, share);
    // (a part whose token is drawn, and what is before it)
    uint32_t token = kNoToken;
    bool again = false;
    for (;;) {
        uint32_t at = kNoToken;
        double goal = 0.0;
        if (total > 0.0) {
            goal = (double)u * total;
            // the first part, then the first token, with which the running sum exceeds the goal; should rounding leave none, the
            // last that has a weight
            uint32_t hit = kNoToken, last = 0;
            double upto = before, hit_before = 0.0, last_before = 0.0;
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k) {
                const double from = upto;
                upto += part[k];
                if (part[k] > 0.0) {
                    last = threadIdx.x * 4u + k + 1u;
                    last_before = from;
                    if (upto > goal && hit == kNoToken) {
                        hit = threadIdx.x * 4u + k;
                        hit_before = from;
                    }
                }
            }
            const uint32_t first = all_min<kWaves>(hit, share), behind = ~all_min<kWaves>(~last, share);
            at = first != kNoToken ? first : behind - 1u;
            if (first != kNoToken ? hit == first : last == behind)
                found_before = first != kNoToken ? hit_before : last_before;
            __syncthreads();
        } else if (again) {
            break;
        }
        if (at == kNoToken) {
            // nothing is left: from p itself
            left.give_up();
            again = true;
            for (uint32_t i = 0; i < parts; ++i) {
                left.part(i, r);
                const double sum = all_sum<kWaves>(r[0] + r[1] + r[2] + r[3], share);
#pragma unroll
                for (uint32_t k = 0; k < 4u; ++k)
                    if (i == threadIdx.x * 4u + k)
                        part[k] = sum;
            }
            before = sum_before<kWaves>(part[0] + part[1] + part[2] + part[3], total, share);
            continue;
        }
        left.part(at, r);
        double all;
        double here = found_before + sum_before<kWaves>(r[0] + r[1] + r[2] + r[3], all, share);
        uint32_t hit = kNoToken, weighty = 0; // (weighty: a token + 1)
#pragma unroll
        for (uint32_t k = 0; k < 4u; ++k) {
            here += r[k];
            if (r[k] > 0.0) {
                weighty = at * kPart + threadIdx.x * 4u + k + 1u;
                if (here > goal && hit == kNoToken)
                    hit = weighty - 1u;
            }
        }
        hit = all_min<kWaves>(hit, share);
        weighty = ~all_min<kWaves>(~weighty, share);
        token = hit != kNoToken ? hit : weighty - 1u;
        break;
    }
    if (threadIdx.x < places)
        d.out_tokens[(uint64_t)b * places + threadIdx.x] = threadIdx.x < stop.accepted ? draft : (threadIdx.x == stop.accepted ? (int32_t)token : -1);
    if (threadIdx.x == 0) {
        d.out_accepted[b] = (int32_t)stop.accepted;
        if (d.seq_len)
            d.out_seq_len[b] = length + (int32_t)stop.accepted + (token != kNoToken);
    }
}

// (as many as run at a time.  More find the place anew, fewer wait longer for their loads: with 1024 the three larger calls above take
// 21.4, 7.7 and 12.8 us, with 2048 14.7, 7.6 and 12.6, with 4096 16.1, 10.2 and 12.6)
constexpr uint32_t kWorkgroups = 2048;
template <class E, class Q>
hipError_t verify(hipStream_t st, const mako_verify_desc& d, const Scratch& sc)
{
    const uint32_t parts = (d.n_vocab + kPart - 1) / kPart;
    const uint32_t each = (uint32_t)min((uint64_t)kMostParts, ((uint64_t)parts * d.n_requests + kWorkgroups - 1) / kWorkgroups);
    const hipError_t e = launch(left_kernel<E, Q>, dim3((parts + each - 1) / each, d.n_requests), kThreads, 0, st, d, sc, each);
    return e != hipSuccess ? e : launch(draw_kernel<E, Q>, dim3(d.n_requests), kThreads, 0, st, d, sc);
}
template <class E>
hipError_t verify(hipStream_t st, const mako_verify_desc& d, const Scratch& sc)
{
    const uint32_t q = d.draft ? d.draft_type : d.target_type;
    return q == MAKO_LOGITS_F32 ? verify<E, F32>(st, d, sc) : (q == MAKO_LOGITS_BF16 ? verify<E, BF16>(st, d, sc) : verify<E, F16>(st, d, sc));
}

} // namespace

hipError_t launch_verify(hipStream_t st, const mako_verify_desc& d, const Scratch& sc)
{
    return d.target_type == MAKO_LOGITS_F32 ? verify<F32>(st, d, sc) : (d.target_type == MAKO_LOGITS_BF16 ? verify<BF16>(st, d, sc) : verify<F16>(st, d, sc));
}

} // namespace step
} // namespace mako
