// Rows' cuts: what temperature, min_p, top_k and top_p leave of a row of logits (mako_step_cut_rows).
//
//   scan_kernel   (k_step_scan.hip) every chunk of every row: its largest logit, its tokens' number, its weights' sum, its first
//                 tokens
//   row_kernel    every row, a workgroup each: the chunks together.  A cut within the chunks' first tokens is found there; one
//                 further down in what a second pass over the row finds around where a sample has it; any other by dividing the
//                 row
//   probs_kernel  where asked for: the rows as probabilities
#include "step_common.h"
#include "step_cut.h"
#include "step_launch.h"

namespace mako {
namespace step {
namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr uint32_t kBins = 1024; // two to a thread
constexpr uint32_t kList = 4096; // tokens that are held in LDS
constexpr uint32_t kSmall = 1024; // ... that are put in order
constexpr uint32_t kWaveList = kList / kWaves; // ... by a wave of a pass over the row
static_assert(kBins == 2 * kThreads, "two bins to a thread");

typedef unsigned long long u64;

struct RowLds {
    uint64_t list[kList];
    uint64_t small[kSmall];
    uint64_t mass[kBins]; // weights in units of 2^-unit
    uint32_t count[kBins];
    float queue[kWaves][128];
    Share<kWaves> share;
    uint32_t n, at, id;
    double m;
    u64 u0, u1;
};

// Where a cut lies: behind the first `rank` tokens, or behind the first whose weights reach `mass`.
struct Want {
    bool by_rank;
    uint32_t rank;
    double mass;
};
struct Cut {
    uint32_t n;  // tokens kept
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

    __device__ __forceinline__ double weigh(float v) const { return weight(v, (double)max, scale); }
    __device__ __forceinline__ u64 units(double w) const { return (u64)rint(ldexp(w, unit)); }
    __device__ __forceinline__ double mass(u64 u) const { return ldexp((double)u, -unit); }
    // (a sum of weights up to `most` keeps below 2^63)
    __device__ __forceinline__ void set_unit(double most) { unit = 62 - ilogb(most); }

    // f(token, logit) for every token of the row
    template <class F>
    __device__ __forceinline__ void each(F f) const
    {
        constexpr uint32_t kStep = kThreads * E::kVec, kAhead = 16 / E::kVec;
        for (uint32_t base = 0; base < n; base += kStep * kAhead) {
            float v[kAhead][E::kVec];
#pragma unroll
            for (uint32_t a = 0; a < kAhead; ++a)
                load_tokens<E>(x, mask, base + a * kStep + threadIdx.x * E::kVec, n, v[a]);
#pragma unroll
            for (uint32_t a = 0; a < kAhead; ++a)
#pragma unroll
                for (uint32_t k = 0; k < E::kVec; ++k)
                    if (v[a][k] > -INFINITY)
                        f(base + a * kStep + threadIdx.x * E::kVec + k, v[a][k]);
        }
    }
};

// Bins between two logits: a function that never falls as the logit does.
struct Bins {
    float top, scale;
    __device__ __forceinline__ Bins(float t, double range) : top(t), scale((float)fmin((double)kBins / fmax(range, 1e-30), 1e30)) {}
    __device__ __forceinline__ uint32_t of(float v) const { return (uint32_t)fminf(fmaxf((top - v) * scale, 0.0f), (float)(kBins - 1u)); }
};

__device__ __forceinline__ void clear_bins(RowLds& lds)
{
    for (uint32_t i = threadIdx.x; i < kBins; i += kThreads) {
        lds.count[i] = 0;
        lds.mass[i] = 0;
    }
    __syncthreads();
}
__device__ __forceinline__ void add_to_bin(RowLds& lds, uint32_t bin, u64 units)
{
    atomicAdd(&lds.count[bin], 1u);
    atomicAdd((u64*)&lds.mass[bin], units);
}

// The first bin with which the running count or mass (of `count` tokens and `mass` before the bins) gets where the cut is; the
// last that has a token, should none get there.  Its number: lds.at, its tokens: lds.n, what lies before it: lds.u0 tokens of
// the bins and lds.u1 units.
template <class E>
__device__ void find_bin(const Row<E>& row, const Want& want, uint32_t count, double mass, RowLds& lds)
{
    const uint32_t a = 2u * threadIdx.x;
    const u64 c[2] = {lds.count[a], lds.count[a + 1]}, m[2] = {lds.mass[a], lds.mass[a + 1]};
    u64 all;
    u64 cb = sum_before<kWaves>(c[0] + c[1], all, lds.share);
    u64 mb = sum_before<kWaves>(m[0] + m[1], all, lds.share);
    const uint32_t last = ~all_min<kWaves>(~(c[1] ? a + 2u : (c[0] ? a + 1u : 0u)), lds.share);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const bool there = c[k] != 0 && (want.by_rank ? count + cb + c[k] >= want.rank : mass + row.mass(mb + m[k]) >= want.mass);
        const bool sooner = cb != 0 && (want.by_rank ? count + cb >= want.rank : mass + row.mass(mb) >= want.mass);
        if ((there && !sooner) || (!there && a + (uint32_t)k + 1u == last)) {
            lds.at = a + (uint32_t)k;
            lds.u0 = cb;
            lds.u1 = mb;
            lds.n = (uint32_t)c[k];
        }
        cb += c[k];
        mb += m[k];
    }
    __syncthreads();
}

__device__ void sort_list(uint64_t* list, uint32_t n)
{
    uint32_t size = 64;
    while (size < n)
        size *= 2;
    for (uint32_t i = n + threadIdx.x; i < size; i += kThreads)
        list[i] = ~0ull;
    __syncthreads();
    for (uint32_t k = 2; k <= size; k *= 2)
        for (uint32_t j = k / 2; j; j /= 2) {
            for (uint32_t t = threadIdx.x; t < size / 2; t += kThreads) {
                const uint32_t i = 2 * t - (t & (j - 1)), l = i + j;
                const uint64_t a = list[i], b = list[l];
                if ((a > b) == ((i & k) == 0)) {
                    list[i] = b;
                    list[l] = a;
                }
            }
            __syncthreads();
        }
}

// The cut in a list of n tokens that holds it, behind `count` tokens of `mass` that come before; the list is put in order.
template <class E>
__device__ Cut cut_in_list(const Row<E>& row, const Want& want, uint64_t* list, uint32_t n, uint32_t count, double mass, RowLds& lds)
{
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
        if (here == kNoToken && (i + 1 == n || (want.by_rank ? count + i + 1 >= want.rank : mass + sum >= want.mass))) {
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

// Bins over lds.list's n tokens, from `top` down by `range`.
template <class E>
__device__ Bins bin_list(const Row<E>& row, uint32_t n, float top, double range, RowLds& lds)
{
    const Bins bins(top, range);
    clear_bins(lds);
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
        const float v = key_logit((uint32_t)(lds.list[i] >> 32));
        add_to_bin(lds, bins.of(v), row.units(row.weigh(v)));
    }
    __syncthreads();
    return bins;
}
// The cut in that list, behind `count` tokens of `mass`.
template <class E>
__device__ Cut cut_in_bins(const Row<E>& row, const Want& want, const Bins& bins, uint32_t n, uint32_t count, double mass, RowLds& lds)
{
    find_bin(row, want, count, mass, lds);
    const uint32_t bin = lds.at, before = (uint32_t)lds.u0, crowd = lds.n;
    const double mass_before = row.mass(lds.u1);
    __syncthreads();
    if (crowd > kSmall) // (the whole list, its bins being of no more use)
        return cut_in_list(row, want, lds.list, n, count, mass, lds);
    if (threadIdx.x == 0)
        lds.n = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
        const uint64_t entry = lds.list[i];
        if (bins.of(key_logit((uint32_t)(entry >> 32))) == bin) {
            const uint32_t at = atomicAdd(&lds.n, 1u);
            if (at < kSmall) // (always: `crowd` of them)
                lds.small[at] = entry;
        }
    }
    __syncthreads();
    return cut_in_list(row, want, lds.small, crowd, count + before, mass + mass_before, lds);
}

// The cut of a row by dividing it: bins over the whole row, a crowded one by its tokens' order keys, digit by digit from the
// top, until few enough are left to hold.  For any row, with a pass over it for every step.
template <class E>
__device__ Cut cut_by_division(Row<E>& row, const Want& want, double total, uint32_t tokens, RowLds& lds)
{
    // over four times what lies between the largest logit and the one of the mean weight
    const Bins bins(row.max, 4.0 * log((double)tokens / total) * kLog2e / row.scale);
    clear_bins(lds);
    row.each([&](uint32_t, float v) { add_to_bin(lds, bins.of(v), row.units(row.weigh(v))); });
    __syncthreads();
    find_bin(row, want, 0, 0.0, lds);
    const uint32_t bin = lds.at;
    uint32_t before = (uint32_t)lds.u0, crowd = lds.n;
    u64 mass_before = lds.u1;
    __syncthreads();
    uint32_t shift = 32, prefix = 0;
    auto in = [&](float v) { return bins.of(v) == bin && (shift == 32u || order_key(v) >> shift == prefix); };
    while (crowd > kList && shift) {
        const uint32_t bits = min(shift, 10u), next = shift - bits;
        clear_bins(lds);
        row.each([&](uint32_t, float v) {
            if (in(v))
                add_to_bin(lds, (order_key(v) >> next) & ((1u << bits) - 1u), row.units(row.weigh(v)));
        });
        __syncthreads();
        find_bin(row, want, before, row.mass(mass_before), lds);
        prefix = (shift == 32u ? 0u : prefix << bits) | lds.at;
        before += (uint32_t)lds.u0;
        mass_before += lds.u1;
        crowd = lds.n;
        shift = next;
        __syncthreads();
    }
    if (crowd > kList) {
        // nothing but equal logits: the cut is behind so many of them, in the tokens' order
        const float v = key_logit(prefix);
        const double w = row.weigh(v);
        uint32_t rank = want.by_rank ? want.rank - before : 0u;
        if (!want.by_rank) {
            const double r = ceil((want.mass - row.mass(mass_before)) / w);
            rank = r >= (double)crowd ? crowd : (r < 1.0 ? 1u : (uint32_t)r);
        }
        uint32_t seen = 0;
        constexpr uint32_t kStep = kThreads * E::kVec;
        for (uint32_t base = 0; base < row.n && seen < rank; base += kStep) {
            float x[E::kVec];
            load_tokens<E>(row.x, row.mask, base + threadIdx.x * E::kVec, row.n, x);
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
            if (at < kList) // (always: `crowd` of them)
                lds.list[at] = (uint64_t)order_key(v) << 32 | id;
        }
    });
    __syncthreads();
    return cut_in_list(row, want, lds.list, crowd, before, row.mass(mass_before), lds);
}

// What a pass over the row finds between two logits, the upper one excluded, and above them.
struct Found {
    uint32_t above, n; // tokens above, and in lds.list; n > kList: more than there is room for
    double side;       // what the tokens above weigh, or those below
};
// The tokens from `low` up to `high` into lds.list; what those above weigh, or those below (`from_above`).  A wave puts the
// tokens in a stretch of the list of its own, and the logits to be weighed in a queue, from which it takes 64 at a time: where
// one logit in ten is weighed, nearly every 64 have one.
template <class E>
__device__ Found look_between(const Row<E>& row, float low, float high, bool from_above, RowLds& lds)
{
    constexpr uint32_t kAhead = 4, kStep = kThreads * E::kVec;
    uint64_t* const list = lds.list + (uint32_t)wave() * kWaveList;
    float* const queue = lds.queue[wave()];
    const u64 lanes_before = (1ull << lane()) - 1ull;
    uint32_t above = 0, n = 0, queued = 0;
    double sum = 0.0;
    for (uint32_t base = 0; base < row.n; base += kStep * kAhead) {
        float v[kAhead][E::kVec];
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a)
            load_tokens<E>(row.x, row.mask, base + a * kStep + threadIdx.x * E::kVec, row.n, v[a]);
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a)
#pragma unroll
            for (uint32_t k = 0; k < E::kVec; ++k) {
                const float x = v[a][k];
                const u64 up = __ballot(x >= high), in = __ballot(x >= low) & ~up;
                const u64 side = from_above ? up : __ballot(x > -INFINITY) & ~(up | in);
                above += (uint32_t)__popcll(up);
                if (in) {
                    const uint32_t at = n + (uint32_t)__popcll(in & lanes_before);
                    if ((in >> lane() & 1ull) && at < kWaveList)
                        list[at] = (uint64_t)order_key(x) << 32 | (base + a * kStep + threadIdx.x * E::kVec + k);
                    n += (uint32_t)__popcll(in);
                }
                if (side) {
                    if (side >> lane() & 1ull)
                        queue[queued + (uint32_t)__popcll(side & lanes_before)] = x;
                    queued += (uint32_t)__popcll(side);
                    if (queued >= 64u) {
                        __builtin_amdgcn_wave_barrier();
                        sum += row.weigh(queue[lane()]);
                        const float rest = queue[64 + lane()];
                        queued -= 64u;
                        __builtin_amdgcn_wave_barrier();
                        if ((uint32_t)lane() < queued)
                            queue[lane()] = rest;
                        __builtin_amdgcn_wave_barrier();
                    }
                }
            }
    }
    __builtin_amdgcn_wave_barrier();
    if ((uint32_t)lane() < queued)
        sum += row.weigh(queue[lane()]);
    // the waves' stretches one after the other
    if (lane() == 0)
        lds.share.u[wave()] = (u64)above << 32 | n;
    uint64_t mine[kWaveList / 64];
#pragma unroll
    for (uint32_t i = 0; i < kWaveList / 64; ++i)
        mine[i] = list[i * 64 + (uint32_t)lane()];
    __syncthreads();
    Found found = {0, 0, 0.0};
    uint32_t place = 0;
    bool room = true;
    for (int w = 0; w < kWaves; ++w) {
        const uint32_t of_wave = (uint32_t)lds.share.u[w];
        room = room && of_wave <= kWaveList;
        if (w == wave())
            place = found.n;
        found.n += of_wave;
        found.above += (uint32_t)(lds.share.u[w] >> 32);
    }
    if (room) {
#pragma unroll
        for (uint32_t i = 0; i < kWaveList / 64; ++i)
            if (i * 64 + (uint32_t)lane() < n)
                lds.list[place + i * 64 + (uint32_t)lane()] = mine[i];
    } else {
        found.n = kList + 1;
    }
    __syncthreads();
    found.side = all_sum<kWaves>(sum, lds.share);
    return found;
}

// The cut by a sample of the row, the first eighth of every chunk: where it says that the cut lies, within three deviations,
// a pass over the row finds the tokens that can be it.  What comes before them is what the pass added up, or the total less
// what lies behind them, whichever are fewer.  false: it is not there after all, or the tokens there are too many.
// (range: of logits, from the largest down, in which the cut is to be expected; total: not where the cut is by rank)
template <class E>
__device__ bool cut_by_sample(const Row<E>& row, const Want& want, double total, uint32_t tokens, double range, Cut& cut, RowLds& lds)
{
    constexpr uint32_t kPer = kChunk / 8, kVecs = kPer / E::kVec, kAhead = 4;
    const Bins bins(row.max, range);
    clear_bins(lds);
    const uint32_t vecs = chunks_of(row.n) * kVecs;
    for (uint32_t base = 0; base < vecs; base += kThreads * kAhead) {
        float v[kAhead][E::kVec];
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a) {
            const uint32_t i = base + a * kThreads + threadIdx.x;
            load_tokens<E>(row.x, row.mask, i < vecs ? i / kVecs * kChunk + i % kVecs * E::kVec : row.n, row.n, v[a]);
        }
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a)
#pragma unroll
            for (uint32_t k = 0; k < E::kVec; ++k)
                if (v[a][k] > -INFINITY)
                    atomicAdd(&lds.count[bins.of(v[a][k])], 1u);
    }
    __syncthreads();
    const uint32_t a = 2 * threadIdx.x;
    const uint32_t c[2] = {lds.count[a], lds.count[a + 1]};
    u64 all;
    uint32_t upto = (uint32_t)sum_before<kWaves>((u64)(c[0] + c[1]), all, lds.share);
    const uint32_t samples = (uint32_t)all;
    if (samples == 0)
        return false;
    const double each = (double)tokens / (double)samples;
    // by rank: tokens of the bins up to this one; by mass: what the tokens behind them weigh.  With the variance of either.
    double behind[2] = {}, var[2] = {};
    if (!want.by_rank) {
        double w[2], sum, sums;
#pragma unroll
        for (int k = 0; k < 2; ++k)
            w[k] = each * row.weigh(bins.top - (float)(((double)(a + k) + 0.5) / (double)bins.scale));
        sum = sum_before<kWaves>(w[0] * c[0] + w[1] * c[1], sums, lds.share);
        behind[0] = sums - sum - w[0] * c[0];
        behind[1] = behind[0] - w[1] * c[1];
        sum = sum_before<kWaves>(w[0] * w[0] * c[0] + w[1] * w[1] * c[1], sums, lds.share);
        var[0] = sums - sum - w[0] * w[0] * c[0];
        var[1] = var[0] - w[1] * w[1] * c[1];
    }
    const double goal = want.by_rank ? (double)want.rank : total - want.mass;
    uint32_t first = kNoToken, last = kNoToken, first_n = 0, last_n = 0;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        upto += c[k];
        const double dev = 3.0 * (want.by_rank ? each * sqrt((double)upto + 1.0) : sqrt(fmax(var[k], 0.0)));
        const double far = want.by_rank ? (double)upto * each - goal : goal - behind[k]; // (grows from bin to bin)
        if (first == kNoToken && far >= -dev) {
            first = a + (uint32_t)k;
            first_n = upto - c[k];
        }
        if (last == kNoToken && far >= dev) {
            last = a + (uint32_t)k;
            last_n = upto;
        }
    }
    const uint32_t first_bin = all_min<kWaves>(first, lds.share), last_bin = all_min<kWaves>(last, lds.share);
    if (first == first_bin)
        lds.u0 = first_n;
    if (last == last_bin)
        lds.u1 = last_n;
    __syncthreads();
    if (first_bin == kNoToken || last_bin >= kBins - 1u) // (the last bin has no lower end)
        return false;
    const uint32_t n_before = (uint32_t)lds.u0, n_bins = (uint32_t)lds.u1 - n_before;
    __syncthreads();
    if ((double)n_bins * each > 0.9 * kList)
        return false;
    const float high = first_bin ? bins.top - (float)((double)first_bin / (double)bins.scale) : INFINITY;
    const float low = bins.top - (float)((double)(last_bin + 1u) / (double)bins.scale);
    const bool from_above = want.by_rank || 2u * (n_before + n_bins / 2u) <= samples;
    const Found found = look_between(row, low, high, from_above, lds);
    if (found.n > kList || found.n == 0)
        return false;
    const float from = fminf(high, row.max);
    const Bins list_bins = bin_list(row, found.n, from, (double)from - (double)low, lds);
    (void)sum_before<kWaves>((u64)lds.mass[a] + lds.mass[a + 1], all, lds.share);
    const double in_list = row.mass(all), mass_before = from_above ? found.side : total - found.side - in_list;
    if (want.by_rank ? found.above >= want.rank || found.above + found.n < want.rank
                     : (found.above != 0 && mass_before >= want.mass) || mass_before + in_list < want.mass)
        return false;
    cut = cut_in_bins(row, want, list_bins, found.n, found.above, mass_before, lds);
    return true;
}

// A row's chunks together: every wave does it by itself, a lane for every 64th chunk.
struct Chunks {
    float max, listed, low;
    uint32_t count, first;
    double total;
    __device__ __forceinline__ Chunks(const ChunkRec* recs, uint32_t chunks, const RowKind& kind) : max(-INFINITY), listed(-INFINITY), low(INFINITY), count(0), first(kNoToken), total(0.0)
    {
        for (uint32_t i = (uint32_t)lane(); i < chunks; i += 64u) {
            const ChunkRec rec = recs[i];
            if (rec.max > max)
                first = rec.first;
            max = fmaxf(max, rec.max);
            listed = fmaxf(listed, rec.listed);
            low = fminf(low, rec.low);
            count += rec.count;
        }
        const float mine = max;
        max = __ockl_wfred_max_f32(max);
        listed = __ockl_wfred_max_f32(listed);
        low = -__ockl_wfred_max_f32(-low);
        count = __ockl_wfred_add_u32(count);
        first = __ockl_wfred_min_u32(mine == max ? first : kNoToken);
        if (kind.sums && count) {
            for (uint32_t i = (uint32_t)lane(); i < chunks; i += 64u)
                if (recs[i].count)
                    total += recs[i].sum * weight(recs[i].max, (double)max, kind.scale);
            total = __ockl_wfred_add_f64(total);
        }
    }
};

// The chunks' first tokens that are the row's, those of logit `listed` and above, into lds.list; how many there are.
__device__ uint32_t gather_lists(const ChunkRec* recs, const uint64_t* lists, uint32_t chunks, float listed, RowLds& lds)
{
    constexpr uint32_t kAhead = 8;
    const uint32_t key = listed > -INFINITY ? order_key(listed + 0.0f) : 0xffffffffu;
    if (threadIdx.x == 0)
        lds.n = 0;
    __syncthreads();
    for (uint32_t base = (uint32_t)wave(); base < chunks; base += kWaves * kAhead) {
        uint64_t entry[kAhead];
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a) {
            const uint32_t c = base + a * kWaves;
            entry[a] = ~0ull;
            if (c < chunks && (uint32_t)lane() < recs[c].n_list)
                entry[a] = lists[c * kChunkList + (uint32_t)lane()];
        }
        u64 in[kAhead];
        uint32_t n = 0;
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a) {
            in[a] = __ballot(entry[a] != ~0ull && (uint32_t)(entry[a] >> 32) <= key);
            n += (uint32_t)__popcll(in[a]);
        }
        uint32_t at = 0;
        if (lane() == 0 && n)
            at = atomicAdd(&lds.n, n);
        at = (uint32_t)__builtin_amdgcn_readfirstlane((int)at);
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a) {
            const uint32_t place = at + (uint32_t)__popcll(in[a] & ((1ull << lane()) - 1ull));
            if ((in[a] >> lane() & 1ull) && place < kList)
                lds.list[place] = entry[a];
            at += (uint32_t)__popcll(in[a]);
        }
    }
    __syncthreads();
    const uint32_t n = lds.n;
    __syncthreads();
    return n;
}

template <class E>
__global__ void __launch_bounds__(kThreads) row_kernel(mako_cut_desc d, Scratch sc)
{
    extern __shared__ unsigned char dyn[];
    RowLds& lds = *reinterpret_cast<RowLds*>(dyn);
    const uint32_t r = blockIdx.x, chunks = chunks_of(d.n_vocab);
    const mako_sampling_params p = d.params[r / d.rows_per_params];
    const RowKind kind(p);
    const ChunkRec* recs = sc.chunks + (uint64_t)r * sc.chunks_cap;
    const Chunks c(recs, chunks, kind);
    mako_row_cut out;
    out.max_logit = c.max;
    out.temperature = kind.greedy ? 0.0f : p.temperature;
    out.cut_logit = -INFINITY;
    out.cut_token = -1;
    out.n_kept = c.count;
    out.total = kind.greedy && c.count ? 1.0 : c.total;
    out.top_token = (int32_t)c.first;
    if (kind.greedy && c.count > 1) {
        out.n_kept = 1;
        out.cut_logit = c.max;
        out.cut_token = out.top_token;
    }
    if (c.count && kind.cut) {
        Row<E> row;
        row.x = static_cast<const typename E::raw*>(d.logits) + (int64_t)r * d.logits_stride;
        row.mask = d.mask ? d.mask + (int64_t)r * d.mask_stride : nullptr;
        row.n = d.n_vocab;
        row.scale = kind.scale;
        row.max = c.max;
        double total = c.total;
        auto add_all = [&]() {
            double mine = 0.0;
            row.each([&](uint32_t, float v) { mine += row.weigh(v); });
            total = all_sum<kWaves>(mine, lds.share);
        };
        const uint32_t n_listed = c.listed < INFINITY ? gather_lists(recs, sc.lists + (uint64_t)r * sc.chunks_cap * kChunkList, chunks, c.listed, lds) : 0u;
        bool list_there = n_listed > 0 && n_listed <= kList;
        // (weights' units: by the total, or, where it is not known, by the most that the list can weigh)
        row.set_unit(kind.sums ? total : (double)max(n_listed, 1u));
        Bins bins(row.max, 1.0);
        double list_mass = 0.0;
        uint32_t rank = kind.top_k ? min(c.count, kind.top_k) : c.count;
        bool all_weighty = !kind.min_p; // (or it is known how many are)
        if (list_there) {
            // (a list of all the row's tokens: the bins go as far down as weights matter)
            bins = bin_list(row, n_listed, row.max, c.listed > -INFINITY ? (double)row.max - (double)c.listed : 64.0 / row.scale, lds);
            u64 all;
            (void)sum_before<kWaves>((u64)lds.mass[2 * threadIdx.x] + lds.mass[2 * threadIdx.x + 1], all, lds.share);
            list_mass = row.mass(all);
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
            uint32_t above = 0;
            row.each([&](uint32_t, float v) { above += row.weigh(v) >= (double)p.min_p; });
            rank = min(rank, max(all_sum<kWaves>(above, lds.share), 1u));
        }
        auto solve = [&](const Want& want) {
            if (list_there && (want.by_rank ? n_listed >= want.rank : list_mass >= want.mass))
                return cut_in_bins(row, want, bins, n_listed, 0, 0.0, lds);
            list_there = false;
            row.set_unit(kind.sums ? total : (double)kList);
            Cut cut;
            if (kind.sums || want.by_rank) {
                // the range: four times what lies between the largest logit and the one of the mean weight, or, where that is not
                // known, twice what the lists reach down
                const double range = kind.sums ? 4.0 * log((double)c.count / total) * kLog2e / row.scale : 2.0 * ((double)row.max - (double)c.listed);
                if (range > 0.0 && range < 1e30 && cut_by_sample(row, want, total, c.count, range, cut, lds))
                    return cut;
            }
            if (total == 0.0)
                add_all();
            row.set_unit(total);
            return cut_by_division(row, want, total, c.count, lds);
        };
        if (rank == c.count && !kind.sums) // (a top_k of no less tokens than there are)
            add_all();
        Cut cut = {c.count, total, 0.0f, 0};
        if (rank < c.count)
            cut = solve(Want{true, rank, 0.0});
        if (kind.top_p)
            cut = solve(Want{false, 0, (double)p.top_p * cut.mass});
        out.total = cut.mass;
        if (cut.n < c.count) {
            out.n_kept = cut.n;
            out.cut_logit = cut.x;
            out.cut_token = (int32_t)cut.id;
        }
    }
    if (threadIdx.x == 0)
        d.out_cuts[r] = out;
}

template <class E>
__global__ void __launch_bounds__(256) probs_kernel(mako_cut_desc d)
{
    const uint32_t r = blockIdx.y;
    const mako_row_cut c = d.out_cuts[r];
    const void* x_row = static_cast<const typename E::raw*>(d.logits) + (int64_t)r * d.logits_stride;
    const uint32_t* mask = d.mask ? d.mask + (int64_t)r * d.mask_stride : nullptr;
    float* out = d.out_probs + (int64_t)r * d.probs_stride;
    const double scale = weight_scale(c.temperature), md = (double)c.max_logit, share = c.total > 0.0 ? 1.0 / c.total : 0.0;
    for (uint32_t j = 0; j < 16u / E::kVec; ++j) {
        const uint32_t i = blockIdx.x * kPart + (j * 256u + threadIdx.x) * E::kVec;
        if (i >= d.n_vocab)
            break;
        float x[E::kVec];
        load_tokens<E>(x_row, mask, i, d.n_vocab, x);
#pragma unroll
        for (uint32_t k = 0; k < E::kVec; ++k) {
            const bool kept = x[k] > c.cut_logit || (x[k] == c.cut_logit && (int32_t)(i + k) <= c.cut_token);
            if (i + k < d.n_vocab)
                out[i + k] = kept ? (float)(weight(x[k], md, scale) * share) : 0.0f;
        }
    }
}

template <class E>
void cut(hipStream_t st, const mako_cut_desc& d, const Scratch& sc)
{
    hipLaunchKernelGGL(row_kernel<E>, dim3(d.n_rows), dim3(kThreads), sizeof(RowLds), st, d, sc);
}
template <class E>
void probs(hipStream_t st, const mako_cut_desc& d)
{
    hipLaunchKernelGGL(probs_kernel<E>, dim3((d.n_vocab + kPart - 1) / kPart, d.n_rows), dim3(256), 0, st, d);
}

} // namespace

hipError_t init_cut()
{
    const void* kernels[] = {reinterpret_cast<const void*>(&row_kernel<F32>), reinterpret_cast<const void*>(&row_kernel<BF16>),
                             reinterpret_cast<const void*>(&row_kernel<F16>)};
    for (const void* k : kernels) {
        const hipError_t e = hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(RowLds));
        if (e != hipSuccess)
            return e;
    }
    return hipSuccess;
}

void launch_cut(hipStream_t st, const mako_cut_desc& d, const Scratch& sc)
{
    launch_scan(st, d, sc);
    d.logits_type == MAKO_LOGITS_F32 ? cut<F32>(st, d, sc) : (d.logits_type == MAKO_LOGITS_BF16 ? cut<BF16>(st, d, sc) : cut<F16>(st, d, sc));
}

void launch_probs(hipStream_t st, const mako_cut_desc& d)
{
    d.logits_type == MAKO_LOGITS_F32 ? probs<F32>(st, d) : (d.logits_type == MAKO_LOGITS_BF16 ? probs<BF16>(st, d) : probs<F16>(st, d));
}

} // namespace step
} // namespace mako
