// Blocks and slots of a paged cache from the requests' lengths (mako_step_assign_blocks).
//
//   blocks_kernel  up to 2048 requests: every workgroup makes the plan for itself (what each request gives back, asks for and is
//                  granted, as running sums in LDS) and does its share of what there is to do: blocks onto the free list and into
//                  tables, tokens' slots
//   counts_kernel  the numbers of blocks, where they replace the ones that the other workgroups' plans are made from
//   plan_kernel, apply_kernel  more requests: the same with one plan, in device memory
//
// Three running sums over the requests (blocks given back, blocks asked for, tokens), and where there is not enough of something
// a second round of sums over those that are still served.  Every output entry then finds its request in them by halving, 11 steps in
// LDS, so that the work is even however lengths differ.  Bound by the launch and a handful of trips to memory: 64 requests of five
// tokens take 4.6 us, 1024 requests with 131072 tokens 7.9 (one plan in device memory and a launch for each half: 10.6 and 18.6),
// 2048 requests of four tokens 8.8, 2049, whose plan is in device memory, 12.6 to 15.3.
#include "step_common.h"
#include "step_launch.h"

namespace mako {
namespace step {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr uint32_t kPlanned = 2048; // requests of a plan in LDS
typedef unsigned long long u64;

// Blocks that a request of these lengths needs; kNone: it is not there (a length below 0), kWide: more than it can have.
constexpr u64 kNone = ~0ull, kWide = ~0ull - 1;
__device__ __forceinline__ u64 blocks_for(const mako_blocks_desc& d, int64_t seq, int64_t more)
{
    if (seq < 0 || more < 0)
        return kNone;
    const u64 want = ((u64)(seq + more) + d.block_size - 1) / d.block_size;
    return want > d.max_blocks || seq + more > INT32_MAX ? kWide : want; // (positions have 31 bits)
}

// For every request what those before it give back and take (n + 1 running sums), the blocks it keeps before it takes any, and
// where its tokens begin (n + 1).  (No sum has more than 31 bits: a batch's tables have no more entries, and tokens that do not
// fit are not laid out.)
struct Plan {
    uint32_t *released, *taken, *held, *start;
    const int32_t* seq;              // the requests' lengths
    uint32_t free_before, available; // blocks on the free list before the call, and with those given back
};

struct PlanLds {
    Share<kWaves> share;
    uint32_t back[kWaves], need[kWaves];
};

// What the threads before this one have of three numbers, and what all have.
struct Three {
    uint32_t back, need;
    u64 tokens;
};
__device__ __forceinline__ Three three_before(const Three& mine, Three& all, PlanLds& lds)
{
    const uint32_t back = __ockl_wfscan_add_u32(mine.back, true), need = __ockl_wfscan_add_u32(mine.need, true);
    const u64 tokens = __ockl_wfscan_add_u64(mine.tokens, true);
    if (lane() == 63) {
        lds.back[wave()] = back;
        lds.need[wave()] = need;
        lds.share.u[wave()] = tokens;
    }
    __syncthreads();
    Three before = {back - mine.back, need - mine.need, tokens - mine.tokens};
    all = {0, 0, 0};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave()) {
            before.back += lds.back[w];
            before.need += lds.need[w];
            before.tokens += lds.share.u[w];
        }
        all.back += lds.back[w];
        all.need += lds.need[w];
        all.tokens += lds.share.u[w];
    }
    __syncthreads();
    return before;
}

// The plan, 1024 requests at a time; `write`: and what the caller gets of it (its numbers of blocks into `counts`, n + 1 of them
// with the free list's behind).
__device__ void make_plan(const mako_blocks_desc& d, Plan& plan, bool write, int32_t* counts, int32_t* n_free, int32_t* seq_copy, PlanLds& lds)
{
    const uint32_t n = d.n_requests;
    plan.free_before = (uint32_t)min(max(*d.n_free, 0), (int32_t)d.free_capacity);
    Three sum = {0, 0, 0}, all;
    for (uint32_t base = 0; base < n; base += kThreads) {
        const uint32_t b = base + threadIdx.x;
        Three mine = {0, 0, 0};
        uint32_t held = 0;
        int32_t status = MAKO_BLOCKS_OK;
        if (b < n) {
            const int32_t seq = d.seq_len[b];
            const int64_t more = d.new_len[b];
            const u64 want = blocks_for(d, seq, more);
            if (seq_copy)
                seq_copy[b] = seq;
            const uint32_t have = (uint32_t)min((int64_t)max(d.n_blocks[b], 0), (int64_t)d.max_blocks);
            held = (uint32_t)min(want, (u64)have);
            mine.back = have - held;
            if (want == kWide)
                status = MAKO_BLOCKS_WIDE;
            else if (want != kNone)
                mine = {mine.back, want > held ? (uint32_t)want - held : 0u, (u64)more};
        }
        const Three before = three_before(mine, all, lds);
        if (b < n) {
            plan.released[b] = sum.back + before.back;
            plan.held[b] = held;
            // (as if all is granted)
            plan.taken[b] = sum.need + before.need;
            plan.start[b] = (uint32_t)(sum.tokens + before.tokens);
            if (write) {
                d.out_status[b] = status;
                d.out_start[b] = (int32_t)(sum.tokens + before.tokens);
                counts[b] = (int32_t)(held + mine.need);
            }
        }
        sum = {sum.back + all.back, sum.need + all.need, sum.tokens + all.tokens};
    }
    plan.available = (uint32_t)min((u64)plan.free_before + sum.back, (u64)d.free_capacity);
    u64 taken = sum.need, tokens = sum.tokens;
    if (sum.need > plan.available || sum.tokens > d.max_tokens) {
        // not all is: request by request in the batch's order
        u64 asked = 0, fitted = 0, total;
        taken = tokens = 0;
        for (uint32_t base = 0; base < n; base += kThreads) {
            const uint32_t b = base + threadIdx.x;
            u64 need = 0, count = 0;
            uint32_t held = 0;
            int32_t status = MAKO_BLOCKS_OK;
            if (b < n) {
                const u64 want = blocks_for(d, d.seq_len[b], d.new_len[b]);
                held = plan.held[b];
                if (want == kWide) {
                    status = MAKO_BLOCKS_WIDE;
                } else if (want != kNone) {
                    count = (u64)d.new_len[b];
                    need = want > held ? want - held : 0;
                }
            }
            const u64 asked_here = asked + sum_before<kWaves>(need, total, lds.share) + need;
            asked += total;
            if (need && asked_here > plan.available)
                status = MAKO_BLOCKS_SHORT;
            if (status)
                count = 0;
            const u64 fit = fitted + sum_before<kWaves>(count, total, lds.share) + count;
            fitted += total;
            if (count && fit > d.max_tokens)
                status = MAKO_BLOCKS_TOKENS;
            if (status)
                need = count = 0;
            const u64 first = tokens + sum_before<kWaves>(count, total, lds.share);
            tokens += total;
            const u64 block = taken + sum_before<kWaves>(need, total, lds.share);
            taken += total;
            if (b < n) {
                plan.taken[b] = (uint32_t)block;
                plan.start[b] = (uint32_t)first;
                if (write) {
                    d.out_status[b] = status;
                    d.out_start[b] = (int32_t)first;
                    counts[b] = (int32_t)(held + need);
                }
            }
        }
    }
    if (threadIdx.x == 0) {
        plan.released[n] = sum.back;
        plan.taken[n] = (uint32_t)taken;
        plan.start[n] = (uint32_t)tokens;
        if (write) {
            d.out_start[n] = (int32_t)tokens;
            *n_free = (int32_t)(plan.available - taken);
        }
    }
}

// The request that entry e is of, by the running sums' n + 1 entries: the last one that begins at or before it.
__device__ __forceinline__ uint32_t owner(const uint32_t* sums, uint32_t n, uint32_t e)
{
    uint32_t low = 0, high = n; // sums[low] <= e < sums[high]
    while (high - low > 1) {
        const uint32_t mid = (low + high) / 2;
        if (sums[mid] <= e)
            low = mid;
        else
            high = mid;
    }
    return low;
}

// One thread's share of what the plan says: entries `from`, `from` + `step` and so on of each kind.
__device__ void apply_plan(const mako_blocks_desc& d, const Plan& plan, uint32_t from, uint32_t step)
{
    const uint32_t n = d.n_requests, tokens = plan.start[n], taken = plan.taken[n];
    // entry e of those that are given back in this call: where it stands in its table (nothing is written there)
    auto given = [&](uint32_t e) {
        const uint32_t b = owner(plan.released, n, e);
        return d.block_table[(int64_t)b * d.table_stride + plan.held[b] + (e - plan.released[b])];
    };
    // the k-th block that is taken: from the top of the list down, what has just been given back first
    auto get = [&](uint32_t k) {
        const uint32_t at = plan.available - 1u - k;
        return at < plan.free_before ? d.free_blocks[at] : given(at - plan.free_before);
    };
    // (the three kinds begin with other threads each: the first entries of all are not one workgroup's)
    for (uint32_t e = (from + step / 3u) % step; e < plan.available - plan.free_before; e += step)
        d.free_blocks[plan.free_before + e] = given(e);
    for (uint32_t k = (from + step / 3u * 2u) % step; k < taken; k += step) {
        const uint32_t b = owner(plan.taken, n, k);
        d.block_table[(int64_t)b * d.table_stride + plan.held[b] + (k - plan.taken[b])] = get(k);
    }
    for (uint32_t t = from; t < d.max_tokens; t += step) {
        int64_t slot = -1;
        uint32_t position = 0;
        int32_t request = -1;
        if (t < tokens) {
            const uint32_t b = owner(plan.start, n, t);
            request = (int32_t)b;
            position = (uint32_t)plan.seq[b] + (t - plan.start[b]);
            const uint32_t at = position / d.block_size, held = plan.held[b];
            // (a block that this call puts into the table is looked up where it comes from)
            const int32_t block = at < held ? d.block_table[(int64_t)b * d.table_stride + at] : get(plan.taken[b] + (at - held));
            slot = (int64_t)block * d.block_size + position % d.block_size;
        }
        d.out_slots[t] = slot;
        if (d.out_positions)
            d.out_positions[t] = (int32_t)position;
        if (d.out_request)
            d.out_request[t] = request;
    }
}

__global__ void __launch_bounds__(kThreads) blocks_kernel(mako_blocks_desc d, int32_t* counts, int32_t* n_free)
{
    __shared__ PlanLds lds;
    __shared__ uint32_t released[kPlanned + 1], taken[kPlanned + 1], held[kPlanned], start[kPlanned + 1];
    __shared__ int32_t seq[kPlanned];
    Plan plan = {released, taken, held, start, seq, 0, 0};
    make_plan(d, plan, blockIdx.x == 0, counts, n_free, seq, lds);
    __syncthreads();
    apply_plan(d, plan, blockIdx.x * kThreads + threadIdx.x, gridDim.x * kThreads);
}

__global__ void __launch_bounds__(256) counts_kernel(mako_blocks_desc d, const int32_t* counts, const int32_t* n_free)
{
    const uint32_t b = blockIdx.x * 256u + threadIdx.x;
    if (b < d.n_requests)
        d.out_n_blocks[b] = counts[b];
    if (b == 0)
        *d.out_n_free = *n_free;
}

__global__ void __launch_bounds__(kThreads) plan_kernel(mako_blocks_desc d, Scratch sc)
{
    __shared__ PlanLds lds;
    Plan plan = {sc.released, sc.taken, sc.held, sc.start, d.seq_len, 0, 0};
    make_plan(d, plan, true, d.out_n_blocks, d.out_n_free, nullptr, lds);
    if (threadIdx.x == 0) {
        sc.free_state[0] = plan.free_before;
        sc.free_state[1] = plan.available;
    }
}

__global__ void __launch_bounds__(256) apply_kernel(mako_blocks_desc d, Scratch sc)
{
    const Plan plan = {sc.released, sc.taken, sc.held, sc.start, d.seq_len, sc.free_state[0], sc.free_state[1]};
    apply_plan(d, plan, blockIdx.x * 256u + threadIdx.x, gridDim.x * 256u);
}

} // namespace

hipError_t launch_blocks(hipStream_t st, const mako_blocks_desc& d, const Scratch& sc)
{
    const uint32_t items = max(d.max_tokens, d.n_requests);
    if (d.n_requests <= kPlanned) {
        // (a workgroup for 1024 tokens.  A call whose numbers of blocks replace the ones it is given has them copied by a launch of
        // their own, unless there is one workgroup alone, which has read them all before it writes any)
        const uint32_t workgroups = min((items + kThreads - 1u) / kThreads, 256u);
        const bool copied = workgroups > 1u && (d.n_blocks == d.out_n_blocks || d.n_free == d.out_n_free);
        int32_t* counts = copied ? reinterpret_cast<int32_t*>(sc.held) : d.out_n_blocks;
        int32_t* n_free = copied ? reinterpret_cast<int32_t*>(sc.free_state) : d.out_n_free;
        const hipError_t e = launch(blocks_kernel, dim3(workgroups), kThreads, 0, st, d, counts, n_free);
        return e != hipSuccess || !copied ? e : launch(counts_kernel, dim3((d.n_requests + 255u) / 256u), 256, 0, st, d, counts, n_free);
    }
    const hipError_t e = launch(plan_kernel, dim3(1), kThreads, 0, st, d, sc);
    return e != hipSuccess ? e : launch(apply_kernel, dim3(min((items + 255u) / 256u, 2048u)), 256, 0, st, d, sc);
}

} // namespace step
} // namespace mako
