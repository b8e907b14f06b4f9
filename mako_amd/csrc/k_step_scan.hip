// The passes over the rows of mako_step_cut_rows: a wave for every chunk of a row, with no word between waves.
//   scan_kernel  every row
//   look_kernel  the rows that have a plan: the tokens around the cut, and what lies above them or below
//
// A chunk is 32 logits a lane, in registers from the one load to the last list entry: the largest, the number, the sum of the
// weights relative to the chunk's own largest (rescaled where the chunks come together) and the list need no second load and no
// barrier.  Bound by vector instructions (80 % of the time), with memory close behind: 512 rows of 129280 bf16 logits (132 MB) 41
// us, some 540 instructions a chunk, most of them without sums, 256 rows of 151552 fp32 logits (155 MB) 43 us, 914 with sums, 20 a
// logit of them for its weight (arithmetic in 64 bits runs at the full rate here).  Chunks of 1024 logits, with as many reductions
// and searches for half the work, took 60 us for both; largest and smallest by instructions that take three logits spill fp32's
// registers (69 us) and gain bf16 nothing.
#include "step_common.h"
#include "step_cut.h"
#include "step_launch.h"

namespace mako {
namespace step {
namespace {

// Bits kHigh to kLow of the n-th largest of the wave's keys, behind those found before (n lanes have a key).
template <int kHigh, int kLow>
__device__ __forceinline__ uint32_t nth_largest(uint32_t key, uint32_t n, uint32_t found)
{
#pragma unroll
    for (int bit = kHigh; bit >= kLow; --bit) {
        const uint32_t trial = found | 1u << bit;
        if ((uint32_t)__popcll(__ballot(key >= trial)) >= n)
            found = trial;
    }
    return found;
}

__device__ __forceinline__ uint32_t lanes_before(unsigned long long lanes)
{
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, 0u));
}

// 64 kEach logits of a row, from token `begin` on; -inf: no token.
template <class E, int kEach>
struct Logits {
    uint32_t begin;
    float x[kEach];

    // (the k-th logit's token)
    __device__ __forceinline__ uint32_t token(int k) const { return begin + ((uint32_t)k / E::kVec * 64u + (uint32_t)lane()) * E::kVec + (uint32_t)k % E::kVec; }

    __device__ __forceinline__ Logits(const mako_cut_desc& d, uint32_t row, uint32_t from) : begin(from)
    {
        const void* x_row = static_cast<const typename E::raw*>(d.logits) + (int64_t)row * d.logits_stride;
        if (begin + 64u * kEach <= d.n_vocab) {
#pragma unroll
            for (int k = 0; k < kEach; k += (int)E::kVec)
                load_whole<E>(x_row, token(k), x + k);
        } else {
#pragma unroll
            for (int k = 0; k < kEach; k += (int)E::kVec)
                load_vec<E>(x_row, token(k), d.n_vocab, x + k);
        }
#pragma unroll
        for (int k = 0; k < kEach; ++k)
            x[k] = fmaxf(x[k], -INFINITY); // (of a NaN and a number, the number)
        if (d.mask) {
            const uint32_t* mask = d.mask + (int64_t)row * d.mask_stride;
#pragma unroll
            for (int k = 0; k < kEach; k += (int)E::kVec) {
                const uint32_t i = token(k), bits = i < d.n_vocab ? mask[i >> 5] >> (i & 31u) : 0u;
#pragma unroll
                for (int e = 0; e < (int)E::kVec; ++e) {
                    const uint32_t keep = (uint32_t)((int32_t)(bits << (31 - e)) >> 31);
                    x[k + e] = __uint_as_float((__float_as_uint(x[k + e]) & keep) | (0xff800000u & ~keep));
                }
            }
        }
    }
    __device__ __forceinline__ void no_infinity()
    {
#pragma unroll
        for (int k = 0; k < kEach; ++k)
            x[k] = fminf(x[k], kFltMax);
    }
    // The lanes' k-th token, of those that have it `in` (the lanes `all`), into a list at `base`.
    __device__ __forceinline__ void put(uint64_t* list, int k, bool in, unsigned long long all, uint32_t base) const
    {
        if (in)
            list[base + lanes_before(all)] = (uint64_t)__float_as_uint(x[k]) << 32 | token(k);
    }
};

template <class E>
__global__ void __launch_bounds__(256, 6) scan_kernel(mako_cut_desc d, Scratch sc)
{
    const uint32_t row = blockIdx.y, chunk = blockIdx.x * 4u + (uint32_t)wave(), chunks = chunks_of(d.n_vocab);
    if (row == 0 && chunk == 0 && lane() == 0)
        *sc.wide = 0;
    if (chunk >= chunks)
        return;
    constexpr int kEach = kChunk / 64;
    Logits<E, kEach> c(d, row, chunk * kChunk);
    const float(&x)[kEach] = c.x;
    const RowKind kind(d.params[row / d.rows_per_params], d.n_vocab);
    float mine = x[0], low = x[0];
#pragma unroll
    for (int k = 1; k < kEach; ++k) {
        mine = fmaxf(mine, x[k]);
        low = fminf(low, x[k]);
    }
    ChunkRec rec = {0.0, -INFINITY, -INFINITY, 0u, 0u, kNoToken, INFINITY};
    rec.max = __ockl_wfred_max_f32(mine);
    if (rec.max == INFINITY) {
        c.no_infinity();
        mine = fminf(mine, kFltMax);
        rec.max = kFltMax;
    }
    const bool full = !__ballot(low == -INFINITY); // nothing but tokens
    if (full) {
        rec.count = kChunk;
    } else {
#pragma unroll
        for (int k = 0; k < kEach; ++k)
            rec.count += (uint32_t)__popcll(__ballot(x[k] > -INFINITY));
    }
    const uint64_t at = (uint64_t)row * sc.chunks_cap + chunk;
    if (rec.count) {
        if (kind.sums) {
            const double md = (double)rec.max;
            double sum = 0.0;
            // (eight at a time: all at once would not leave the logits in registers)
#pragma unroll
            for (int k = 0; k < kEach; ++k) {
                sum += weight(x[k], md, kind.scale);
                if (k % 8 == 7)
                    __builtin_amdgcn_sched_barrier(0);
            }
            rec.sum = __ockl_wfred_add_f64(sum);
        }
        if (kind.min_p) {
            if (!full) {
                low = INFINITY;
#pragma unroll
                for (int k = 0; k < kEach; ++k)
                    low = fminf(low, x[k] > -INFINITY ? x[k] : INFINITY);
            }
            rec.low = -__ockl_wfred_max_f32(-low);
        }
        if (kind.cut && d.n_vocab > kWholeRow) {
            // The chunk's first tokens: those not below the n-th largest of the lanes' largest, to 16 bits of their order; where these
            // are too many, to all bits, then those above it (equal ones), then of half as many lanes.  A chunk of few tokens lists
            // them all.
            uint64_t* list = sc.lists + at * kChunkList;
            const bool all_listed = rec.count <= kChunkList;
            const uint32_t key = ~order_key(mine); // (rises with the logit)
            uint32_t n = min(kind.list_length(chunks), (uint32_t)__popcll(__ballot(mine > -INFINITY)));
            uint32_t found = nth_largest<31, 16>(key, n, 0u);
            rec.listed = all_listed ? -kFltMax : key_logit(~found);
#pragma unroll 1
            for (uint32_t tries = 0;; ++tries) {
                rec.n_list = 0;
#pragma unroll
                for (int k = 0; k < kEach; ++k) {
                    const bool in = x[k] >= rec.listed;
                    const unsigned long long all = __ballot(in);
                    if (all) {
                        const uint32_t more = (uint32_t)__popcll(all);
                        if (rec.n_list + more <= kChunkList)
                            c.put(list, k, in, all, rec.n_list);
                        rec.n_list += more;
                    }
                }
                if (rec.n_list <= kChunkList)
                    break;
                if (tries % 2u == 0) {
                    n = tries ? n / 2u : n;
                    if (n == 0) {
                        rec.listed = INFINITY;
                        rec.n_list = 0;
                        break;
                    }
                    found = nth_largest<15, 0>(key, n, tries ? nth_largest<31, 16>(key, n, 0u) : found);
                    rec.listed = key_logit(~found);
                } else {
                    rec.listed = key_logit(order_key(rec.listed + 0.0f) - 1u); // (all of the next larger number and above)
                }
            }
            if (all_listed)
                rec.listed = -INFINITY;
        } else {
#pragma unroll
            for (int k = kEach - 1; k >= 0; --k)
                if (x[k] == rec.max)
                    rec.first = c.token(k);
            rec.first = __ockl_wfred_min_u32(rec.first);
        }
    }
    rec.max += 0.0f;
    if (lane() == 0)
        sc.chunks[at] = rec;
}

template <class E>
__global__ void __launch_bounds__(256, 6) look_kernel(mako_cut_desc d, Scratch sc)
{
    constexpr int kEach = 16; // (a chunk in two halves: the more waves, the less they wait for)
    __shared__ float weighed[4][64 * kEach];
    const uint32_t chunks = chunks_of(d.n_vocab), groups = (chunks + 3) / 4;
    for (uint32_t item = blockIdx.x; item < d.n_rows * groups; item += gridDim.x) {
        // (the plan is asked for before it is known that there is one)
        const uint32_t at_plan = item / groups, chunk = item % groups * 4u + (uint32_t)wave();
        const RowPlan plan = sc.plans[at_plan];
        if (at_plan >= *sc.wide)
            return;
        const uint32_t row = plan.row;
        const float low = plan.low, high = plan.high, max = plan.max;
        const double scale = plan.scale;
        const bool from_above = plan.from_above;
        if (!plan.look || chunk >= chunks)
            continue;
        ChunkRec rec = {0.0, 0.0f, 0.0f, 0u, 0u, 0u, 0.0f};
        // (what is weighed moves together first: where it is one logit in ten, nearly every 64 have one)
        float* const mine = weighed[wave()];
        const uint64_t at = (uint64_t)at_plan * sc.chunks_cap + chunk;
        uint64_t* list = sc.looks + at * kLookList;
        double sum = 0.0;
#pragma unroll 1
        for (uint32_t begin = chunk * kChunk; begin < min((chunk + 1u) * kChunk, d.n_vocab); begin += 64u * kEach) {
            Logits<E, kEach> c(d, row, begin);
            if (max == kFltMax)
                c.no_infinity();
            uint32_t n = 0;
#pragma unroll
            for (int k = 0; k < kEach; ++k) {
                const float x = c.x[k];
                const bool up = x >= high, in = x >= low && !up, weigh = from_above ? up : x < low && x > -INFINITY;
                const unsigned long long all = __ballot(in), side = __ballot(weigh);
                rec.count += (uint32_t)__popcll(__ballot(up));
                if (all) {
                    const uint32_t more = (uint32_t)__popcll(all);
                    if (rec.n_list + more <= kLookList)
                        c.put(list, k, in, all, rec.n_list);
                    rec.n_list += more;
                }
                if (side) {
                    if (weigh)
                        mine[n + lanes_before(side)] = x;
                    n += (uint32_t)__popcll(side);
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll 1
            for (uint32_t i = (uint32_t)lane(); i < n; i += 64u)
                sum += weight<true>(mine[i], (double)max, scale);
            __builtin_amdgcn_wave_barrier();
        }
        rec.sum = __ockl_wfred_add_f64(sum);
        if (lane() == 0)
            sc.chunks[at] = rec;
    }
}

template <class E>
hipError_t scan(hipStream_t st, const mako_cut_desc& d, const Scratch& sc)
{
    return launch(scan_kernel<E>, dim3((chunks_of(d.n_vocab) + 3) / 4, d.n_rows), 256, 0, st, d, sc);
}

constexpr uint32_t kLookWorkgroups = 4096; // (256 wide rows of 151552 take 111 us in all, with 2048 114, with 8192 112)
template <class E>
hipError_t look(hipStream_t st, const mako_cut_desc& d, const Scratch& sc)
{
    const uint32_t items = d.n_rows * ((chunks_of(d.n_vocab) + 3) / 4); // (65535 rows of 256 at most)
    return launch(look_kernel<E>, dim3(items < kLookWorkgroups ? items : kLookWorkgroups), 256, 0, st, d, sc);
}

} // namespace

hipError_t launch_scan(hipStream_t st, const mako_cut_desc& d, const Scratch& sc)
{
    return d.logits_type == MAKO_LOGITS_F32 ? scan<F32>(st, d, sc) : (d.logits_type == MAKO_LOGITS_BF16 ? scan<BF16>(st, d, sc) : scan<F16>(st, d, sc));
}

hipError_t launch_look(hipStream_t st, const mako_cut_desc& d, const Scratch& sc)
{
    return d.logits_type == MAKO_LOGITS_F32 ? look<F32>(st, d, sc) : (d.logits_type == MAKO_LOGITS_BF16 ? look<BF16>(st, d, sc) : look<F16>(st, d, sc));
}

} // namespace step
} // namespace mako
