// Rows' cuts: what temperature, min_p, top_k and top_p leave of a row of logits (mako_step_cut_rows).
//
//   scan_kernel   (k_step_scan.hip) every chunk of every row: its largest logit, its tokens' number, its weights' sum, its first
//                 tokens
//   row_kernel    every row, a workgroup each: the chunks together, and a cut that lies within their first tokens.  For any other
//                 a plan: where the cut has to be, by a sample of the row
//   look_kernel   (k_step_scan.hip) the rows that have a plan: the tokens there, and what lies above them, or below
//   wide_kernel   these rows, a workgroup each: the cut among those tokens, or, should it not be there, by dividing the row
//   probs_kernel  where asked for: the rows as probabilities
//
// The mathematics: with the weights w = exp((x - max) / T), a row's cut is the place in the order of falling logits behind a rank
// (min_p and top_k come down to one) or behind the least number of tokens that weigh top_p of all.  No row is sorted: the pass
// over it leaves some 10 to 71 of every 2048 tokens, among which a narrow cut lies; a wide one is guessed by a sample of an
// eighth of the row, and a second pass collects the tokens around it and adds up those above.  Among at most 6144 tokens, in LDS,
// 1024 bins of logits say which bin holds it, and the bin's tokens are counted against each other.  Weights are 64-bit floats, and
// where they are added up in an order that chance makes (bins, atomics) whole numbers of a unit, so that results do not vary.
//
// What bounds them: 64 rows of 129280 fp32 logits (33.1 MB), some cut beyond their lists, take 43 us: scan 12.9 (2.6 TB/s), row 13.9,
// look 8.0, wide 10.4; one row of 151552 34: 5.4, 12.5, 7.4, 9.0; 256 of them, half of them flat, 96: 42 (3.7 TB/s, vector
// instructions 78 % of the time), 15, 24 (6.4 TB/s, from the Infinity Cache) and 14.5.  row_kernel and wide_kernel are chains of some
// fifteen trips to memory, LDS and barriers with one workgroup's latency in each, their code read from memory as they go (a pass
// fewer through the list, with the exponentials in more places, took 1 us longer).
#include "step_common.h"
#include "step_cut.h"
#include "step_launch.h"

namespace mako {
namespace step {
namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64; // two workgroups to a CU, by LDS
constexpr uint32_t kBins = 1024;  // two to a thread
constexpr uint32_t kList = kWholeRow; // tokens that are held in LDS
constexpr uint32_t kSmall = 1024; // ... of a bin
constexpr uint32_t kCrowd = 256;  // ... that are counted against each other; more are sorted
static_assert(kBins == 2 * kThreads, "two bins to a thread");
constexpr int kTries = 3; // how wide a guess may be

typedef unsigned long long u64;

struct RowLds {
    uint64_t list[kList];
    uint64_t small[kSmall];
    uint64_t crowd[kCrowd];
    u64 small_units[kCrowd];
    u64 mass[kBins]; // weights in units of 2^-unit
    uint32_t count[kBins];
    uint32_t ids[kBins];
    Share<kWaves> share;
    uint32_t counts[kWaves];
    double squares[kWaves];
    uint32_t first_bin[kTries], last_bin[kTries], n_before[kTries], n_upto[kTries];
    uint32_t n, at, before, id, first;
    u64 mass_before;
    double m;
};

// Where a cut lies: behind the first `rank` tokens, or (rank 0) behind the first whose weights reach `mass`.
struct Want {
    uint32_t rank;
    double mass;
    __device__ __forceinline__ bool reached(uint32_t n, double m) const { return rank ? n >= rank : m >= mass; }
};
struct Cut {
    uint32_t n;  // tokens kept; 0: not found
    double mass; // and what they weigh
    float x;     // the last of them
    uint32_t id;
};

// What the passes over a row need to know of it.
template <class E>
struct Row {
    const void* x;
    const uint32_t* mask;
    uint32_t n;
    float max;
    double scale; // of weights
    int unit;     // weights are added up as whole multiples of 2^-unit, in any order

    __device__ __forceinline__ Row(const mako_cut_desc& d, uint32_t r, float largest, double weights)
        : x(static_cast<const typename E::raw*>(d.logits) + (int64_t)r * d.logits_stride), mask(d.mask ? d.mask + (int64_t)r * d.mask_stride : nullptr), n(d.n_vocab),
          max(largest), scale(weights), unit(0)
    {
    }
    __device__ __forceinline__ double weigh(float v) const { return weight(v, (double)max, scale); }
    __device__ __forceinline__ u64 units(double w) const { return (u64)rint(ldexp(w, unit)); }
    __device__ __forceinline__ double mass(u64 u) const { return ldexp((double)u, -unit); }
    // (a sum of weights up to `most` keeps below 2^63)
    __device__ __forceinline__ void set_unit(double most) { unit = 63 - __builtin_amdgcn_frexp_exp(most); }

    // f(token, logit) for every token of the row
    template <class F>
    __device__ __forceinline__ void each(F f) const
    {
        constexpr uint32_t kStep = kThreads * E::kVec, kAhead = 16 / E::kVec;
        for (uint32_t base = 0; base < n; base += kStep * kAhead) {
            float v[kAhead][E::kVec];
            load_tokens<E>(x, mask, [&](uint32_t a) { return base + a * kStep + threadIdx.x * E::kVec; }, n, v);
#pragma unroll
            for (uint32_t a = 0; a < kAhead; ++a)
#pragma unroll
                for (uint32_t k = 0; k < E::kVec; ++k)
                    if (v[a][k] > -INFINITY)
                        f(base + a * kStep + threadIdx.x * E::kVec + k, v[a][k]);
        }
    }
    __device__ __forceinline__ double add_all(RowLds& lds) const
    {
        double mine = 0.0;
        each([&](uint32_t, float v) { mine += weigh(v); });
        return all_sum<kWaves>(mine, lds.share);
    }
};

// Bins between two logits: a function that never falls as the logit does.
struct Bins {
    float top, scale;
    __device__ __forceinline__ Bins(float t, float range) : top(t), scale(fminf((float)kBins / fmaxf(range, 1e-30f), 1e30f)) {}
    __device__ __forceinline__ uint32_t of(float v) const { return (uint32_t)fminf(fmaxf((top - v) * scale, 0.0f), (float)(kBins - 1u)); }
};

__device__ __forceinline__ void clear_bins(RowLds& lds)
{
    for (uint32_t i = threadIdx.x; i < kBins; i += kThreads) {
        lds.count[i] = 0;
        lds.mass[i] = 0;
    }
}
__device__ __forceinline__ void add_to_bin(RowLds& lds, uint32_t bin, u64 units)
{
    atomicAdd(&lds.count[bin], 1u);
    atomicAdd(&lds.mass[bin], units);
}

// The first bin with which the running count and mass get where the cut is, behind `count` tokens; what these and some of the bins'
// tokens weigh is mass(the latter's units, the units of all in the bins).
struct Bin {
    uint32_t at, before, n; // n 0: none does.  before: tokens in the bins before it
    u64 mass_before, all;   // and their weights' units, and those of all
};
template <class E, class F>
__device__ __forceinline__ Bin find_bin(const Row<E>& row, const Want& want, uint32_t count, F mass, RowLds& lds)
{
    const uint32_t a = 2u * threadIdx.x;
    const uint32_t c[2] = {lds.count[a], lds.count[a + 1]};
    const u64 m[2] = {lds.mass[a], lds.mass[a + 1]};
    const uint32_t c_wave = __ockl_wfscan_add_u32(c[0] + c[1], true);
    const u64 m_wave = __ockl_wfscan_add_u64(m[0] + m[1], true);
    if (lane() == 63) {
        lds.counts[wave()] = c_wave;
        lds.share.u[wave()] = m_wave;
    }
    if (threadIdx.x == 0)
        lds.n = 0;
    __syncthreads();
    uint32_t cb = c_wave - c[0] - c[1];
    u64 mb = m_wave - m[0] - m[1], all = 0;
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave()) {
            cb += lds.counts[w];
            mb += lds.share.u[w];
        }
        all += lds.share.u[w];
    }
    bool was = cb != 0 && want.reached(count + cb, mass(mb, all));
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const bool is = want.reached(count + cb + c[k], mass(mb + m[k], all));
        if (c[k] != 0 && is && !was) {
            lds.at = a + (uint32_t)k;
            lds.before = cb;
            lds.mass_before = mb;
            lds.n = c[k];
        }
        cb += c[k];
        mb += m[k];
        was = cb != 0 && is;
    }
    __syncthreads();
    const Bin bin = {lds.at, lds.before, lds.n, lds.mass_before, all};
    __syncthreads();
    return bin;
}

__device__ __forceinline__ void sort_list(uint64_t* list, uint32_t n)
{
    uint32_t size = 64;
    while (size < n)
        size *= 2;
    // (the largest list has no room to be made a power of two long: what lies behind it is not touched, and counts as largest)
    for (uint32_t k = 2; k <= size; k *= 2)
        for (uint32_t j = k / 2; j; j /= 2) {
            // (every pair in rising order: in the first step of a round the upper half is read backwards)
            for (uint32_t t = threadIdx.x; t < size / 2; t += kThreads) {
                const uint32_t low = t & (j - 1), i = 2 * t - low, l = j == k / 2 ? i + 2 * j - 1 - 2 * low : i + j;
                if (l < n) {
                    const uint64_t a = list[i], b = list[l];
                    if (a > b) {
                        list[i] = b;
                        list[l] = a;
                    }
                }
            }
            __syncthreads();
        }
}

// How many of n equal tokens are before the cut, behind `count` tokens of `mass`; it is within them.
__device__ __forceinline__ uint32_t rank_of_equals(const Want& want, uint32_t n, uint32_t count, double mass, double w)
{
    if (want.rank)
        return want.rank - count;
    const double r = ceil((want.mass - mass) / w);
    return r >= (double)n ? n : (r < 1.0 ? 1u : (uint32_t)r);
}

// The cut in a list of n tokens that holds it, behind `count` tokens of `mass` that come before.
template <class E>
__device__ __forceinline__ Cut cut_in_list(const Row<E>& row, const Want& want, uint64_t* list, uint32_t n, uint32_t count, double mass, RowLds& lds)
{
    // many equal logits (of 16 bits, most): the cut is behind so many of them, in the tokens' order
    const uint32_t key = (uint32_t)(list[0] >> 32);
    bool equal = n > 32u;
    if (equal) {
        for (uint32_t i = threadIdx.x; i < n; i += kThreads)
            equal = equal && (uint32_t)(list[i] >> 32) == key;
        for (uint32_t i = threadIdx.x; i < kBins; i += kThreads)
            lds.ids[i] = 0;
        equal = all_min<kWaves>(equal, lds.share);
    }
    if (equal) {
        const float v = key_logit(key);
        const double w = row.weigh(v);
        const uint32_t rank = rank_of_equals(want, n, count, mass, w);
        const uint32_t shift = row.n > kBins ? 22u - (uint32_t)__builtin_clz(row.n - 1u) : 0u; // (tokens to bins)
        for (uint32_t i = threadIdx.x; i < n; i += kThreads)
            atomicAdd(&lds.ids[(uint32_t)list[i] >> shift], 1u);
        if (threadIdx.x == 0)
            lds.n = 0;
        __syncthreads();
        const uint32_t a = 2 * threadIdx.x, c[2] = {lds.ids[a], lds.ids[a + 1]};
        u64 all;
        uint32_t before = (uint32_t)sum_before<kWaves>((u64)(c[0] + c[1]), all, lds.share);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (before < rank && rank <= before + c[k]) {
                lds.at = a + (uint32_t)k;
                lds.before = before;
            }
            before += c[k];
        }
        __syncthreads();
        const uint32_t bin = lds.at, in_bin = rank - lds.before;
        for (uint32_t i = threadIdx.x; i < n; i += kThreads)
            if ((uint32_t)list[i] >> shift == bin) {
                const uint32_t at = atomicAdd(&lds.n, 1u);
                lds.ids[at] = (uint32_t)list[i]; // (a bin has 1024 tokens at most, of 2^20)
            }
        __syncthreads();
        const uint32_t crowd = lds.n;
        for (uint32_t i = threadIdx.x; i < crowd; i += kThreads) {
            uint32_t place = 0;
            for (uint32_t j = 0; j < crowd; ++j)
                place += lds.ids[j] <= lds.ids[i];
            if (place == in_bin)
                lds.id = lds.ids[i];
        }
        __syncthreads();
        const Cut cut = {count + rank, mass + (double)rank * w, v, lds.id};
        __syncthreads();
        return cut;
    }
    if (n <= kCrowd) {
        // every token's place, and what those up to it weigh, by a look at all the others: no order needs to be made
        // (eight at a time, in an array that is filled up with what is behind all)
        uint64_t mine = ~0ull;
        if (threadIdx.x < kCrowd) {
            if (threadIdx.x < n)
                mine = list[threadIdx.x];
            lds.crowd[threadIdx.x] = mine;
            lds.small_units[threadIdx.x] = threadIdx.x < n ? row.units(row.weigh(key_logit((uint32_t)(mine >> 32)))) : 0ull;
        }
        if (threadIdx.x == 0)
            lds.at = kNoToken;
        __syncthreads();
        uint32_t place = 0;
        u64 upto = 0;
        if (threadIdx.x < ((n + 63u) & ~63u)) {
            for (uint32_t i = 0; i < n; i += 8u)
#pragma unroll
                for (uint32_t k = 0; k < 8u; ++k) {
                    const bool before = lds.crowd[i + k] <= mine && i + k < n;
                    place += before;
                    upto += before ? lds.small_units[i + k] : 0ull;
                }
            if (threadIdx.x < n && (place == n || want.reached(count + place, mass + row.mass(upto))))
                atomicMin(&lds.at, place);
        }
        __syncthreads();
        if (threadIdx.x < n && place == lds.at) {
            lds.id = threadIdx.x;
            lds.m = mass + row.mass(upto);
        }
        __syncthreads();
        const uint64_t last = list[lds.id];
        const Cut cut = {count + lds.at, lds.m, key_logit((uint32_t)(last >> 32)), (uint32_t)last};
        __syncthreads();
        return cut;
    }
    sort_list(list, n);
    // (a stretch of the list to each thread)
    const uint32_t each = (n + kThreads - 1) / kThreads, from = min(threadIdx.x * each, n), to = min(from + each, n);
    double mine = 0.0, all;
    for (uint32_t i = from; i < to; ++i)
        mine += row.weigh(key_logit((uint32_t)(list[i] >> 32)));
    double sum = sum_before<kWaves>(mine, all, lds.share);
    uint32_t here = kNoToken;
    double here_mass = 0.0;
    for (uint32_t i = from; i < to; ++i) {
        sum += row.weigh(key_logit((uint32_t)(list[i] >> 32)));
        if (here == kNoToken && (i + 1 == n || want.reached(count + i + 1, mass + sum))) {
            here = i;
            here_mass = mass + sum;
        }
    }
    const uint32_t first = all_min<kWaves>(here, lds.share);
    if (here == first)
        lds.m = here_mass;
    __syncthreads();
    const uint64_t last = list[first];
    const Cut cut = {count + first + 1u, lds.m, key_logit((uint32_t)(last >> 32)), (uint32_t)last};
    __syncthreads();
    return cut;
}

// Bins (cleared) over lds.list's n tokens.
template <class E>
__device__ __forceinline__ void bin_list(const Row<E>& row, const Bins& bins, uint32_t n, RowLds& lds)
{
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
        const float v = key_logit((uint32_t)(lds.list[i] >> 32));
        add_to_bin(lds, bins.of(v), row.units(row.weigh(v)));
    }
    __syncthreads();
}
// The cut in that list, behind `count` tokens of `mass`: in one of its bins.
template <class E>
__device__ __forceinline__ Cut cut_in_bin(const Row<E>& row, const Want& want, const Bins& bins, const Bin& bin, uint32_t n, uint32_t count, double mass, RowLds& lds)
{
    if (bin.n > kSmall)
        return cut_in_list(row, want, lds.list, n, count, mass, lds);
    if (threadIdx.x == 0)
        lds.n = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
        const uint64_t entry = lds.list[i];
        if (bins.of(key_logit((uint32_t)(entry >> 32))) == bin.at) {
            const uint32_t at = atomicAdd(&lds.n, 1u);
            if (at < kSmall) // (always: bin.n of them)
                lds.small[at] = entry;
        }
    }
    __syncthreads();
    return cut_in_list(row, want, lds.small, bin.n, count + bin.before, mass + row.mass(bin.mass_before), lds);
}

// The cut in that list, if it is there, with nothing before it.
template <class E>
__device__ __forceinline__ Cut cut_in_bins(const Row<E>& row, const Want& want, const Bins& bins, uint32_t n, RowLds& lds)
{
    const Bin bin = find_bin(row, want, 0u, [&](u64 upto, u64) { return row.mass(upto); }, lds);
    if (bin.n == 0)
        return {0, 0.0, 0.0f, 0};
    return cut_in_bin(row, want, bins, bin, n, 0u, 0.0, lds);
}

// The range of logits, from the largest down, in which a cut by mass is to be expected: four times what lies between the largest
// and the one of the mean weight.
__device__ __forceinline__ float range_of(uint32_t tokens, double total, double scale)
{
    return 4.0f * __builtin_amdgcn_logf((float)tokens * __builtin_amdgcn_rcpf((float)total)) / (float)fmin(scale, 1e30);
}

// The cut of a row by dividing it: bins over the whole row, a crowded one by its tokens' order keys, digit by digit from the
// top, until few enough are left to hold.  For any row, with a pass over it for every step.
template <class E>
__device__ __forceinline__ Cut cut_by_division(Row<E>& row, const Want& want, double total, uint32_t tokens, RowLds& lds)
{
    row.set_unit(total);
    const Bins bins(row.max, range_of(tokens, total, row.scale));
    clear_bins(lds);
    __syncthreads();
    // (the last bin: in a row of few heavy tokens, most)
    uint32_t last_n = 0;
    u64 last_units = 0;
    row.each([&](uint32_t, float v) {
        const uint32_t at = bins.of(v);
        const u64 units = row.units(row.weigh(v));
        if (at < kBins - 1u) {
            add_to_bin(lds, at, units);
        } else {
            ++last_n;
            last_units += units;
        }
    });
    if (last_n) {
        atomicAdd(&lds.count[kBins - 1u], last_n);
        atomicAdd(&lds.mass[kBins - 1u], last_units);
    }
    __syncthreads();
    Bin bin = find_bin(row, want, 0, [&](u64 upto, u64) { return row.mass(upto); }, lds);
    if (bin.n == 0) // (all the row's tokens, as whole units, weigh less than is wanted of their sum: nothing is cut off)
        return {tokens, total, 0.0f, 0};
    const uint32_t first = bin.at;
    uint32_t before = bin.before;
    u64 mass_before = bin.mass_before;
    uint32_t shift = 32, prefix = 0;
    auto in = [&](float v) { return bins.of(v) == first && (shift == 32u || order_key(v) >> shift == prefix); };
    while (bin.n > kList && shift) {
        const uint32_t bits = min(shift, 10u), next = shift - bits;
        clear_bins(lds);
        __syncthreads();
        row.each([&](uint32_t, float v) {
            if (in(v))
                add_to_bin(lds, (order_key(v) >> next) & ((1u << bits) - 1u), row.units(row.weigh(v)));
        });
        __syncthreads();
        // (one of them: what weighs enough up to the end of the bin that is divided does so up to the last of its parts, since both are
        // the same whole number of units, made a mass once.  As a sum of two masses it can be a bit less)
        bin = find_bin(row, want, before, [&](u64 upto, u64) { return row.mass(mass_before + upto); }, lds);
        prefix = (shift == 32u ? 0u : prefix << bits) | bin.at;
        before += bin.before;
        mass_before += bin.mass_before;
        shift = next;
    }
    if (bin.n > kList) {
        // nothing but equal logits: the cut is behind so many of them, in the tokens' order
        const float v = key_logit(prefix);
        const double w = row.weigh(v);
        const uint32_t rank = rank_of_equals(want, bin.n, before, row.mass(mass_before), w);
        uint32_t seen = 0;
        constexpr uint32_t kStep = kThreads * E::kVec;
        for (uint32_t base = 0; base < row.n && seen < rank; base += kStep) {
            float v1[1][E::kVec];
            load_tokens<E>(row.x, row.mask, [&](uint32_t) { return base + threadIdx.x * E::kVec; }, row.n, v1);
            const float(&x)[E::kVec] = v1[0];
            uint32_t mine = 0;
#pragma unroll
            for (uint32_t k = 0; k < E::kVec; ++k)
                mine += x[k] == v;
            u64 all;
            uint32_t at = seen + (uint32_t)sum_before<kWaves>((u64)mine, all, lds.share);
#pragma unroll
            for (uint32_t k = 0; k < E::kVec; ++k)
                if (x[k] == v && ++at == rank)
                    lds.id = base + threadIdx.x * E::kVec + k;
            seen += (uint32_t)all;
        }
        __syncthreads();
        const Cut cut = {before + rank, row.mass(mass_before) + (double)rank * w, v, lds.id};
        __syncthreads();
        return cut;
    }
    if (threadIdx.x == 0)
        lds.n = 0;
    __syncthreads();
    row.each([&](uint32_t id, float v) {
        if (in(v)) {
            const uint32_t at = atomicAdd(&lds.n, 1u);
            if (at < kList) // (always: bin.n of them)
                lds.list[at] = (uint64_t)order_key(v) << 32 | id;
        }
    });
    __syncthreads();
    return cut_in_list(row, want, lds.list, bin.n, before, row.mass(mass_before), lds);
}

// A guess where the cut of a row lies, by a sample of it, an eighth of every chunk in kPieces places (128 bytes of fp32 each): within
// four deviations, and where these hold too many tokens, within three, or two and a half.  (7 of row_kernel's 12.5 us on one row of 151552, 4 of them
// the sample; a sixteenth took as long, with longer lists for wide_kernel.  In one place the times are the same, but rows whose
// tokens stand in order are guessed wrongly and divided: 290 us instead of 76.)
// (range: of logits, from the largest down, in which the cut is to be expected; total: not where the cut is by rank)
struct Guess {
    float low, high;
    uint32_t from_above, look;
};
template <class E>
__device__ __forceinline__ Guess guess(const Row<E>& row, const Want& want, double total, uint32_t tokens, float range, RowLds& lds)
{
    constexpr uint32_t kPieces = 8, kPiece = kChunk / kPieces, kVecs = kPiece / 8u / E::kVec, kAhead = 40 / E::kVec;
    const Guess none = {0.0f, 0.0f, 0u, 0u};
    const Bins bins(row.max, range);
    clear_bins(lds);
    __syncthreads();
    uint32_t below = 0; // (in the last bin: in a row of few heavy tokens, most)
    const uint32_t vecs = (row.n + kPiece - 1u) / kPiece * kVecs;
    for (uint32_t base = 0; base < vecs; base += kThreads * kAhead) {
        float v[kAhead][E::kVec];
        auto at = [&](uint32_t a) {
            const uint32_t i = base + a * kThreads + threadIdx.x;
            return i < vecs ? i / kVecs * kPiece + i % kVecs * E::kVec : row.n;
        };
        load_tokens<E>(row.x, row.mask, at, row.n, v);
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a)
#pragma unroll
            for (uint32_t k = 0; k < E::kVec; ++k)
                if (v[a][k] > -INFINITY) {
                    const uint32_t bin = bins.of(v[a][k]);
                    if (bin < kBins - 1u)
                        atomicAdd(&lds.count[bin], 1u);
                    else
                        ++below;
                }
    }
    below = __ockl_wfred_add_u32(below);
    if (lane() == 0 && below)
        atomicAdd(&lds.count[kBins - 1u], below);
    __syncthreads();
    // running sums of the bins, by rank of their tokens alone, by mass of what these weigh and of its squares too
    const uint32_t a = 2 * threadIdx.x;
    const uint32_t c[2] = {lds.count[a], lds.count[a + 1]};
    double w[2] = {}, sum = 0.0, squares = 0.0;
    const float step = __builtin_amdgcn_rcpf(bins.scale); // (of logits, a bin)
    if (!want.rank) {
        const float step_log2 = (float)(row.scale * (double)step);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            w[k] = (double)__builtin_amdgcn_exp2f(-((float)(a + (uint32_t)k) + 0.5f) * step_log2);
            sum += w[k] * c[k];
            squares += w[k] * w[k] * c[k];
        }
        sum = __ockl_wfscan_add_f64(sum, true);
        squares = __ockl_wfscan_add_f64(squares, true);
    }
    uint32_t upto = __ockl_wfscan_add_u32(c[0] + c[1], true);
    if (lane() == 63) {
        lds.counts[wave()] = upto;
        lds.share.d[wave()] = sum;
        lds.squares[wave()] = squares;
    }
    if (threadIdx.x == 0)
        for (int tries = 0; tries < kTries; ++tries)
            lds.first_bin[tries] = lds.last_bin[tries] = 0;
    __syncthreads();
    uint32_t samples = 0, n_all = 0;
    double sums = 0.0, sum_all = 0.0, squares_before = 0.0, squares_all = 0.0;
    for (int v = 0; v < kWaves; ++v) {
        if (v == wave()) {
            n_all = samples;
            sum_all = sums;
            squares_before = squares_all;
        }
        samples += lds.counts[v];
        sums += lds.share.d[v];
        squares_all += lds.squares[v];
    }
    if (samples == 0)
        return none;
    upto += n_all;
    sum += sum_all;
    squares += squares_before;
    // how far behind the cut a bin's end is (it grows from bin to bin), and the deviation of that: by rank in tokens up to there,
    // by mass in what the tokens behind it weigh.  (A sample that holds one of the row's few heavy tokens has both far off in the
    // bins up to it.)  The cut is behind the last bin whose end is surely before it, and in the one behind the last whose end may be
    // before it, or sooner.
    const float each = (float)tokens * __builtin_amdgcn_rcpf((float)samples);
    const double behind_goal = total - want.mass;
    double behind = sums - sum, var = squares_all - squares;
    // (a small rank: few samples say little where tokens of like logits stand together)
    const float margin = want.rank && want.rank < kListTopK ? 512.0f : 0.0f;
    uint32_t n = upto, first[kTries] = {}, last[kTries] = {};
#pragma unroll
    for (int k = 1; k >= 0; --k) {
        const float far = want.rank ? (float)n * each - (float)want.rank : (float)(behind_goal - behind * (double)each);
        const float dev = each * __builtin_amdgcn_sqrtf(want.rank ? (float)n + 1.0f : (float)fmax(var, 0.0));
#pragma unroll
        for (int tries = 0; tries < kTries; ++tries) {
            const float z = tries == 0 ? 4.0f : (tries == 1 ? 3.0f : 2.5f);
            if (far < -z * dev)
                first[tries] = max(first[tries], a + (uint32_t)k + 1u);
            if (far < z * dev || (far < z * dev + margin && a + (uint32_t)k + 1u < kBins - 1u))
                last[tries] = max(last[tries], a + (uint32_t)k + 1u);
        }
        n -= c[k];
        behind += w[k] * c[k];
        var += w[k] * w[k] * c[k];
    }
#pragma unroll
    for (int tries = 0; tries < kTries; ++tries) {
        first[tries] = __ockl_wfred_max_u32(first[tries]);
        last[tries] = __ockl_wfred_max_u32(last[tries]);
        if (lane() == 0) {
            atomicMax(&lds.first_bin[tries], first[tries]);
            atomicMax(&lds.last_bin[tries], last[tries]);
        }
    }
    __syncthreads();
#pragma unroll
    for (int tries = 0; tries < kTries; ++tries) {
        n = upto - c[0] - c[1];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (a + (uint32_t)k == lds.first_bin[tries])
                lds.n_before[tries] = n;
            n += c[k];
            if (a + (uint32_t)k == lds.last_bin[tries])
                lds.n_upto[tries] = n;
        }
    }
    __syncthreads();
    for (int tries = 0; tries < kTries; ++tries) {
        const uint32_t first_bin = lds.first_bin[tries], last_bin = lds.last_bin[tries];
        if (last_bin >= kBins - 1u) // (the last bin has no lower end)
            return none;
        const uint32_t n_before = lds.n_before[tries], n_bins = lds.n_upto[tries] - n_before;
        if ((float)n_bins * each > 0.9f * kList)
            continue;
        const float low = bins.top - (float)(last_bin + 1u) * step;
        // (a rank that there is room for has all tokens up to it listed: a top_p behind it is then found among them)
        if (want.rank && (float)lds.n_upto[tries] * each <= 0.9f * kList)
            return {low, INFINITY, 1u, 1u};
        return {low, first_bin ? bins.top - (float)first_bin * step : INFINITY, want.rank || 2u * n_before + n_bins <= samples, 1u};
    }
    return none;
}

// A row's chunks together: every wave does it by itself, a lane for every 64th chunk.
constexpr uint32_t kHeld = 2; // of a lane's chunks that are in registers
struct Chunks {
    ChunkRec rec[kHeld];
    float max, listed, low;
    uint32_t count, first;
    double total;

    __device__ __forceinline__ void load(const ChunkRec* recs, uint32_t chunks)
    {
#pragma unroll
        for (uint32_t h = 0; h < kHeld; ++h) {
            rec[h] = {0.0, -INFINITY, -INFINITY, 0u, 0u, kNoToken, INFINITY};
            if (h * 64u + (uint32_t)lane() < chunks)
                rec[h] = recs[h * 64u + (uint32_t)lane()];
        }
    }
    __device__ __forceinline__ void join(const ChunkRec* recs, uint32_t chunks, const RowKind& kind)
    {
        max = listed = -INFINITY;
        low = INFINITY;
        count = 0;
        first = kNoToken;
        total = 0.0;
        auto add = [&](const ChunkRec& one) {
            if (one.max > max)
                first = one.first;
            max = fmaxf(max, one.max);
            listed = fmaxf(listed, one.listed);
            low = fminf(low, one.low);
            count += one.count;
        };
#pragma unroll
        for (uint32_t h = 0; h < kHeld; ++h)
            add(rec[h]);
        for (uint32_t i = kHeld * 64u + (uint32_t)lane(); i < chunks; i += 64u)
            add(recs[i]);
        const float mine = max;
        max = __ockl_wfred_max_f32(max);
        listed = __ockl_wfred_max_f32(listed);
        count = __ockl_wfred_add_u32(count);
        first = __ockl_wfred_min_u32(mine == max ? first : kNoToken);
        if (kind.min_p)
            low = -__ockl_wfred_max_f32(-low);
        if (kind.sums && count) {
#pragma unroll
            for (uint32_t h = 0; h < kHeld; ++h)
                if (rec[h].count)
                    total += rec[h].sum * weight(rec[h].max, (double)max, kind.scale);
            for (uint32_t i = kHeld * 64u + (uint32_t)lane(); i < chunks; i += 64u)
                if (recs[i].count)
                    total += recs[i].sum * weight(recs[i].max, (double)max, kind.scale);
            total = __ockl_wfred_add_f64(total);
        }
    }
};

// The chunks' lists, kSlots lanes to a chunk: their first kSlots tokens, of as many chunks as fit kAhead loads, are asked for
// together with the chunks' records, whatever their number is.
template <uint32_t kSlots, uint32_t kRoom, uint32_t kAhead>
struct Lists {
    static constexpr uint32_t kOfWave = 64 / kSlots, kOfAll = kOfWave * kWaves; // chunks of a load
    static_assert(kOfAll <= 64 && kAhead * kOfAll <= kHeld * 64u && kHeld == 2 && kAhead >= 4, "chunks that are in registers");
    uint64_t entry[kAhead];

    static __device__ __forceinline__ uint32_t chunk(uint32_t a) { return a * kOfAll + (uint32_t)wave() * kOfWave + (uint32_t)lane() / kSlots; }

    __device__ __forceinline__ void load(const uint64_t* lists, uint32_t chunks)
    {
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a) {
            entry[a] = 0;
            if (chunk(a) < chunks)
                entry[a] = lists[chunk(a) * kRoom + (uint32_t)lane() % kSlots];
        }
    }
    // The tokens of logits from `from` on into lds.list (lds.n is 0), and the first of those of logit `max` into lds.first; how
    // many there are, which may be more than there is room for.
    __device__ __forceinline__ uint32_t gather(const Chunks& c, const ChunkRec* recs, const uint64_t* lists, uint32_t chunks, float from, float max, RowLds& lds) const
    {
        const u64 before = (1ull << lane()) - 1ull;
        auto put = [&](uint64_t e, bool in, uint32_t place) {
            const float x = __uint_as_float((uint32_t)(e >> 32));
            if (in && x == max)
                atomicMin(&lds.first, (uint32_t)e);
            if (in && place < kList)
                lds.list[place] = (uint64_t)order_key(x + 0.0f) << 32 | (uint32_t)e;
        };
        u64 in[kAhead];
        uint32_t n = 0;
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a) {
            const uint32_t of_chunk = (uint32_t)__shfl((int)c.rec[a * kOfAll / 64u].n_list, (int)(chunk(a) & 63u));
            in[a] = __ballot(chunk(a) < chunks && (uint32_t)lane() % kSlots < of_chunk && __uint_as_float((uint32_t)(entry[a] >> 32)) >= from);
            n += (uint32_t)__popcll(in[a]);
        }
        uint32_t at = 0;
        if (lane() == 0 && n)
            at = atomicAdd(&lds.n, n);
        at = (uint32_t)__builtin_amdgcn_readfirstlane((int)at);
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a) {
            put(entry[a], in[a] >> lane() & 1ull, at + (uint32_t)__popcll(in[a] & before));
            at += (uint32_t)__popcll(in[a]);
        }
        // longer lists, and the chunks beyond: every wave those of every eighth chunk, of four of them at a time
        constexpr uint32_t kHeldChunks = kAhead * kOfAll, kBatch = 4;
        if (chunks > kHeldChunks || __ballot(c.rec[0].n_list > kSlots || c.rec[1].n_list > kSlots))
            for (uint32_t base = (uint32_t)wave(); base < chunks; base += kWaves * kBatch) {
                uint32_t of_chunk[kBatch], slot[kBatch];
                bool more = false;
#pragma unroll
                for (uint32_t a = 0; a < kBatch; ++a) {
                    const uint32_t i = base + a * kWaves;
                    of_chunk[a] = 0;
                    if (i < 64u * kHeld)
                        of_chunk[a] = (uint32_t)__builtin_amdgcn_readlane((int)(i < 64u ? c.rec[0].n_list : c.rec[1].n_list), (int)(i & 63u));
                    else if (i < chunks)
                        of_chunk[a] = recs[i].n_list;
                    slot[a] = i < kHeldChunks ? kSlots : 0u;
                    more = more || slot[a] < of_chunk[a];
                }
                while (more) {
                    uint64_t e[kBatch];
                    uint32_t m = 0;
                    more = false;
#pragma unroll
                    for (uint32_t a = 0; a < kBatch; ++a) {
                        e[a] = (uint64_t)__float_as_uint(-INFINITY) << 32;
                        if (slot[a] + (uint32_t)lane() < of_chunk[a])
                            e[a] = lists[(base + a * kWaves) * kRoom + slot[a] + (uint32_t)lane()];
                    }
#pragma unroll
                    for (uint32_t a = 0; a < kBatch; ++a) {
                        in[a] = __ballot(slot[a] + (uint32_t)lane() < of_chunk[a] && __uint_as_float((uint32_t)(e[a] >> 32)) >= from);
                        m += (uint32_t)__popcll(in[a]);
                        slot[a] += 64u;
                        more = more || slot[a] < of_chunk[a];
                    }
                    at = 0;
                    if (lane() == 0 && m)
                        at = atomicAdd(&lds.n, m);
                    at = (uint32_t)__builtin_amdgcn_readfirstlane((int)at);
#pragma unroll
                    for (uint32_t a = 0; a < kBatch; ++a) {
                        put(e[a], in[a] >> lane() & 1ull, at + (uint32_t)__popcll(in[a] & before));
                        at += (uint32_t)__popcll(in[a]);
                    }
                }
            }
        __syncthreads();
        const uint32_t all = lds.n;
        __syncthreads();
        return all;
    }
};
using FirstLists = Lists<32, kChunkList, 5>; // (80 chunks: vocabularies of up to 163 840)
using LookLists = Lists<64, kLookList, 10>;

__device__ __forceinline__ void store_cut(mako_row_cut& out, const Cut& cut, uint32_t tokens)
{
    if (threadIdx.x == 0) {
        out.total = cut.mass;
        if (cut.n < tokens) {
            out.n_kept = cut.n;
            out.cut_logit = cut.x;
            out.cut_token = (int32_t)cut.id;
        }
    }
}

template <class E>
__global__ void __launch_bounds__(kThreads, 4) row_kernel(mako_cut_desc d, Scratch sc)
{
    extern __shared__ unsigned char dyn[];
    RowLds& lds = *reinterpret_cast<RowLds*>(dyn);
    const uint32_t r = blockIdx.x, chunks = chunks_of(d.n_vocab);
    const ChunkRec* recs = sc.chunks + (uint64_t)r * sc.chunks_cap;
    const uint64_t* lists = sc.lists + (uint64_t)r * sc.chunks_cap * kChunkList;
    Chunks c;
    c.load(recs, chunks);
    // (before the row's parameters are known: a row that is not cut has no lists, and what is there is not looked at)
    FirstLists listed;
    const bool whole = d.n_vocab <= kWholeRow;
    if (!whole)
        listed.load(lists, chunks);
    const mako_sampling_params p = d.params[r / d.rows_per_params];
    const RowKind kind(p, d.n_vocab);
    if (kind.cut) {
        clear_bins(lds);
        if (threadIdx.x == 0) {
            lds.n = 0;
            lds.first = kNoToken;
        }
    }
    c.join(recs, chunks, kind);
    Row<E> row(d, r, c.max, kind.scale);
    uint32_t first = c.first, n_listed = 0;
    if (kind.cut && c.count) {
        __syncthreads();
        if (whole) {
            row.each([&](uint32_t id, float v) { lds.list[atomicAdd(&lds.n, 1u)] = (uint64_t)order_key(v) << 32 | id; });
            __syncthreads();
            n_listed = c.count;
            c.listed = -INFINITY;
        } else {
            if (c.listed < INFINITY)
                n_listed = listed.gather(c, recs, lists, chunks, c.listed, c.max, lds);
            first = lds.first;
            if (first == kNoToken) { // (too many equal ones for any list)
                __syncthreads();
                row.each([&](uint32_t id, float v) {
                    if (v == c.max)
                        atomicMin(&lds.first, id);
                });
                __syncthreads();
                first = lds.first;
            }
        }
    }
    mako_row_cut& out = d.out_cuts[r];
    if (threadIdx.x == 0) {
        mako_row_cut plain;
        plain.total = kind.greedy && c.count ? 1.0 : c.total;
        plain.max_logit = c.max;
        plain.temperature = kind.greedy ? 0.0f : p.temperature;
        plain.n_kept = kind.greedy ? min(c.count, 1u) : c.count;
        plain.top_token = (int32_t)first;
        plain.cut_logit = plain.n_kept < c.count ? c.max : -INFINITY;
        plain.cut_token = plain.n_kept < c.count ? plain.top_token : -1;
        out = plain;
    }
    if (!kind.cut || c.count == 0)
        return;
    const bool list_there = n_listed > 0 && n_listed <= kList;
    // (weights' units: by the total, or, where it is not known, by the most that the list can weigh)
    row.set_unit(kind.sums ? c.total : (double)max(n_listed, 1u));
    // (a list of all the row's tokens: the bins go as far down as weights matter)
    const Bins bins(row.max, c.listed > -INFINITY ? row.max - c.listed : (float)(64.0 / row.scale));
    // (no token weighs more than the first, which weighs 1)
    const bool none_weighty = kind.min_p && p.min_p > 1.0f;
    uint32_t rank = none_weighty ? 1u : (kind.top_k ? min(c.count, kind.top_k) : c.count);
    bool all_weighty = none_weighty || !kind.min_p; // (or it is known how many are)
    if (list_there) {
        bin_list(row, bins, n_listed, lds);
        if (kind.min_p) {
            uint32_t above = 0;
            for (uint32_t i = threadIdx.x; i < n_listed; i += kThreads)
                above += row.weigh(key_logit((uint32_t)(lds.list[i] >> 32))) >= (double)p.min_p;
            above = all_sum<kWaves>(above, lds.share);
            if (above < n_listed || n_listed == c.count || rank <= n_listed) {
                rank = min(rank, max(above, 1u));
                all_weighty = true;
            }
        }
    }
    if (!all_weighty && row.weigh(c.low) < (double)p.min_p) {
        // the least logit that weighs enough, between the smallest, which does not, and the largest, by halving their order keys
        uint32_t enough = order_key(row.max), less = order_key(c.low);
        while (less - enough > 1u) {
            const uint32_t middle = enough + (less - enough) / 2u;
            if (row.weigh(key_logit(middle)) >= (double)p.min_p)
                enough = middle;
            else
                less = middle;
        }
        const float least = key_logit(enough);
        uint32_t above = 0;
        row.each([&](uint32_t, float v) { above += v >= least; });
        rank = min(rank, max(all_sum<kWaves>(above, lds.share), 1u));
    }
    Cut cut = {c.count, c.total, 0.0f, 0};
    if (rank == c.count) {
        if (!kind.sums) { // (a top_k of no less tokens than there are: they are listed, unless they stand together)
            if (list_there && n_listed == c.count) {
                u64 all;
                (void)sum_before<kWaves>(lds.mass[2 * threadIdx.x] + lds.mass[2 * threadIdx.x + 1], all, lds.share);
                cut.mass = row.mass(all);
            } else {
                cut.mass = row.add_all(lds);
            }
        }
    } else {
        cut.n = 0;
        if (list_there && rank <= n_listed)
            cut = cut_in_bins(row, Want{rank, 0.0}, bins, n_listed, lds);
    }
    Want want = {0u, 0.0};
    if (cut.n == 0) {
        want.rank = rank;
    } else if (kind.top_p) {
        want.mass = (double)p.top_p * cut.mass;
        cut.n = 0;
        if (list_there)
            cut = cut_in_bins(row, want, bins, n_listed, lds);
    }
    if (cut.n) {
        store_cut(out, cut, c.count);
        return;
    }
    // the cut lies further down
    // (a cut by rank may be far from where the weight is: twice what the lists reach down)
    const float range = fmaxf(kind.sums ? range_of(c.count, c.total, row.scale) : 0.0f, want.rank ? 2.0f * (row.max - c.listed) : 0.0f);
    Guess where = {0.0f, 0.0f, 0u, 0u};
    if ((kind.sums || want.rank) && range > 0.0f && range < 1e30f)
        where = guess(row, want, c.total, c.count, range, lds);
    if (threadIdx.x == 0) {
        RowPlan& plan = sc.plans[atomicAdd(sc.wide, 1u)];
        plan.mass = want.mass;
        plan.total = c.total;
        plan.rank = want.rank;
        plan.row = r;
        plan.tokens = c.count;
        plan.max = row.max;
        plan.scale = row.scale;
        plan.low = where.low;
        plan.high = where.high;
        plan.top_p = kind.top_p ? p.top_p : 1.0f;
        plan.sums = kind.sums;
        plan.from_above = where.from_above;
        plan.look = where.look;
    }
}

template <class E>
__global__ void __launch_bounds__(kThreads, 4) wide_kernel(mako_cut_desc d, Scratch sc)
{
    extern __shared__ unsigned char dyn[];
    RowLds& lds = *reinterpret_cast<RowLds*>(dyn);
    const uint32_t chunks = chunks_of(d.n_vocab);
    for (uint32_t i = blockIdx.x; i < d.n_rows; i += gridDim.x) {
        const RowPlan plan = sc.plans[i];
        if (i >= *sc.wide)
            return;
        // (what the pass around the cut found is asked for before the plan is there)
        const ChunkRec* recs = sc.chunks + (uint64_t)i * sc.chunks_cap;
        const uint64_t* lists = sc.looks + (uint64_t)i * sc.chunks_cap * kLookList;
        Chunks c;
        LookLists listed;
        c.load(recs, chunks);
        listed.load(lists, chunks);
        mako_row_cut& out = d.out_cuts[plan.row];
        Row<E> row(d, plan.row, plan.max, plan.scale);
        Want want = {plan.rank, plan.mass};
        Cut cut = {0, 0.0, 0.0f, 0};
        double total = plan.total;
        Bins list_bins(row.max, 1.0f);
        uint32_t listed_n = 0; // tokens in lds.list, where the cut is
        float low = plan.low, high = plan.high;
        __syncthreads();
        clear_bins(lds);
        if (threadIdx.x == 0)
            lds.n = 0;
        row.set_unit(plan.sums ? total : (double)kList);
        if (plan.look) {
            double side = 0.0;
            uint32_t above = 0, n = 0;
            bool room = true;
            auto add = [&](const ChunkRec& one) {
                side += one.sum;
                above += one.count;
                n += one.n_list;
                room = room && one.n_list <= kLookList;
            };
#pragma unroll
            for (uint32_t h = 0; h < kHeld; ++h)
                if (h * 64u + (uint32_t)lane() < chunks)
                    add(c.rec[h]);
            for (uint32_t k = kHeld * 64u + (uint32_t)lane(); k < chunks; k += 64u)
                add(recs[k]);
            side = __ockl_wfred_add_f64(side);
            above = __ockl_wfred_add_u32(above);
            n = __ockl_wfred_add_u32(n);
            room = !__ballot(!room) && n <= kList;
            __syncthreads();
            if (room) {
                (void)listed.gather(c, recs, lists, chunks, -INFINITY, INFINITY, lds);
                const float from = fminf(high, row.max);
                list_bins = Bins(from, from - low);
                bin_list(row, list_bins, n, lds);
                auto before = [&](u64 all) { return plan.from_above ? side : total - side - row.mass(all); };
                const Bin bin = find_bin(row, want, above, [&](u64 upto, u64 all) { return before(all) + row.mass(upto); }, lds);
                if (above && want.reached(above, before(bin.all))) {
                    const float width = from - low;
                    low = high;
                    high += 2.0f * width;
                } else if (bin.n) {
                    cut = cut_in_bin(row, want, list_bins, bin, n, above, before(bin.all), lds);
                    listed_n = n;
                } else {
                    high = low;
                    low -= 2.0f * (from - low);
                }
            }
            if (cut.n == 0) {
                // Too many tokens for a chunk's list (they stand together), or the cut is beside them: in a pass over the row by this
                // workgroup alone, there.  (One row in some thousands: 40 us, a division of a row of 129280 takes 100 and more.)
                u64 units = 0, all;
                above = 0;
                clear_bins(lds);
                if (threadIdx.x == 0)
                    lds.n = 0;
                __syncthreads();
                row.each([&](uint32_t id, float v) {
                    if (v >= high) {
                        ++above;
                        units += row.units(row.weigh(v));
                    } else if (v >= low) {
                        const uint32_t at = atomicAdd(&lds.n, 1u);
                        if (at < kList)
                            lds.list[at] = (uint64_t)order_key(v) << 32 | id;
                    }
                });
                above = all_sum<kWaves>(above, lds.share);
                (void)sum_before<kWaves>(units, all, lds.share);
                n = lds.n;
                __syncthreads();
                if (n <= kList) {
                    const double weight_above = row.mass(all);
                    const float from = fminf(high, row.max);
                    list_bins = Bins(from, from - low);
                    bin_list(row, list_bins, n, lds);
                    const Bin bin = find_bin(row, want, above, [&](u64 upto, u64) { return weight_above + row.mass(upto); }, lds);
                    if (bin.n && !(above && want.reached(above, weight_above))) {
                        cut = cut_in_bin(row, want, list_bins, bin, n, above, weight_above, lds);
                        listed_n = n;
                    }
                }
            }
        }
        if (cut.n == 0) {
            if (!plan.sums)
                total = row.add_all(lds);
            cut = cut_by_division(row, want, total, plan.tokens, lds);
        }
        if (plan.rank && plan.top_p < 1.0f) {
            want = Want{0, (double)plan.top_p * cut.mass};
            cut.n = 0;
            if (listed_n && high == INFINITY)
                cut = cut_in_bins(row, want, list_bins, listed_n, lds);
            if (cut.n == 0) {
                if (!plan.sums && total == 0.0)
                    total = row.add_all(lds);
                cut = cut_by_division(row, want, total, plan.tokens, lds);
            }
        }
        store_cut(out, cut, plan.tokens);
    }
}

constexpr uint32_t kProbs = 2048; // logits of a workgroup (of 128 rows of 32000 it takes 9.4 us; 1024: 9.6; 4096, with a branch for each logit: 10.5)
template <class E>
__global__ void __launch_bounds__(256) probs_kernel(mako_cut_desc d)
{
    const uint32_t r = blockIdx.y;
    const mako_row_cut c = d.out_cuts[r];
    const void* x_row = static_cast<const typename E::raw*>(d.logits) + (int64_t)r * d.logits_stride;
    const uint32_t* mask = d.mask ? d.mask + (int64_t)r * d.mask_stride : nullptr;
    float* out = d.out_probs + (int64_t)r * d.probs_stride;
    const double scale = weight_scale(c.temperature), md = (double)c.max_logit, share = c.total > 0.0 ? 1.0 / c.total : 0.0;
    // (all of a thread's logits asked for before the first is used; four at a time, so that a wave's stores leave no gaps)
    constexpr uint32_t kFours = kProbs / 1024u;
    const uint32_t first = blockIdx.x * kProbs + threadIdx.x * 4u;
    float x[kFours][4];
#pragma unroll
    for (uint32_t j = 0; j < kFours; ++j) {
        const uint32_t i = first + j * 1024u;
        load_four<E>(x_row, i, d.n_vocab, x[j]);
        const uint32_t bits = !mask ? 0xfu : (i < d.n_vocab ? mask[i >> 5] >> (i & 31u) : 0u);
#pragma unroll
        for (uint32_t k = 0; k < 4u; ++k)
            x[j][k] = token_logit(x[j][k], (bits >> k) & 1u);
    }
#pragma unroll
    for (uint32_t j = 0; j < kFours; ++j) {
        const uint32_t i = first + j * 1024u;
        if (i >= d.n_vocab)
            break;
        float p[4] = {};
        bool kept[4], any = false;
#pragma unroll
        for (uint32_t k = 0; k < 4u; ++k) {
            kept[k] = x[j][k] > c.cut_logit || (x[j][k] == c.cut_logit && (int32_t)(i + k) <= c.cut_token);
            any = any || kept[k];
        }
        if (__ballot(any)) {
            double t[4], w[4];
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k)
                t[k] = ((double)x[j][k] - md) * scale;
            exp2_down<4>(t, w);
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k)
                p[k] = kept[k] ? (float)(w[k] * share) : 0.0f;
        }
        if (i + 4u <= d.n_vocab) {
            const words_at_4 w = {__float_as_uint(p[0]), __float_as_uint(p[1]), __float_as_uint(p[2]), __float_as_uint(p[3])};
            *reinterpret_cast<words_at_4*>(out + i) = w;
        } else {
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k)
                if (i + k < d.n_vocab)
                    out[i + k] = p[k];
        }
    }
}

constexpr uint32_t kWideWorkgroups = 512; // (two to a CU: what fits; 512 wide rows of 32000 take 75 us in all, with 256 workgroups 82)
template <class E>
hipError_t cut(hipStream_t st, const mako_cut_desc& d, const Scratch& sc)
{
    hipError_t e = launch_scan(st, d, sc);
    if (e == hipSuccess)
        e = launch(row_kernel<E>, dim3(d.n_rows), kThreads, sizeof(RowLds), st, d, sc);
    if (d.n_vocab <= kWholeRow)
        return e; // (every row's tokens are listed: its cut is found there)
    if (e == hipSuccess)
        e = launch_look(st, d, sc);
    if (e == hipSuccess)
        e = launch(wide_kernel<E>, dim3(d.n_rows < kWideWorkgroups ? d.n_rows : kWideWorkgroups), kThreads, sizeof(RowLds), st, d, sc);
    return e;
}
template <class E>
hipError_t probs(hipStream_t st, const mako_cut_desc& d)
{
    return launch(probs_kernel<E>, dim3((d.n_vocab + kProbs - 1) / kProbs, d.n_rows), 256, 0, st, d);
}

} // namespace

hipError_t init_cut()
{
    const void* kernels[] = {reinterpret_cast<const void*>(&row_kernel<F32>),  reinterpret_cast<const void*>(&row_kernel<BF16>),
                             reinterpret_cast<const void*>(&row_kernel<F16>),  reinterpret_cast<const void*>(&wide_kernel<F32>),
                             reinterpret_cast<const void*>(&wide_kernel<BF16>), reinterpret_cast<const void*>(&wide_kernel<F16>)};
    for (const void* k : kernels) {
        const hipError_t e = hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(RowLds));
        if (e != hipSuccess)
            return e;
    }
    return hipSuccess;
}

hipError_t launch_cut(hipStream_t st, const mako_cut_desc& d, const Scratch& sc)
{
    return d.logits_type == MAKO_LOGITS_F32 ? cut<F32>(st, d, sc) : (d.logits_type == MAKO_LOGITS_BF16 ? cut<BF16>(st, d, sc) : cut<F16>(st, d, sc));
}

hipError_t launch_probs(hipStream_t st, const mako_cut_desc& d)
{
    return d.logits_type == MAKO_LOGITS_F32 ? probs<F32>(st, d) : (d.logits_type == MAKO_LOGITS_BF16 ? probs<BF16>(st, d) : probs<F16>(st, d));
}

} // namespace step
} // namespace mako
