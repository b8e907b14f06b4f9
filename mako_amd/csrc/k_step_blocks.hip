// Blocks and slots of a paged cache from the requests' lengths (mako_step_assign_blocks).
//
//   plan_kernel   one workgroup: what every request gives back, asks for and is granted, as running sums
//   apply_kernel  as many as there are tokens for: blocks onto the free list and into tables, tokens' slots
#include "step_common.h"
#include "step_launch.h"

namespace mako {
namespace step {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
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

__global__ void __launch_bounds__(kThreads) plan_kernel(mako_blocks_desc d, Scratch sc)
{
    __shared__ Share<kWaves> share;
    const uint32_t n = d.n_requests, capacity = d.free_capacity;
    const uint32_t free_before = (uint32_t)min(max(*d.n_free, 0), (int32_t)capacity);
    u64 released = 0, asked = 0, fitted = 0, taken = 0, tokens = 0, all;
    // first what is given back: the requests of a tile of 1024 at a time
    for (uint32_t base = 0; base < n; base += kThreads) {
        const uint32_t b = base + threadIdx.x;
        u64 back = 0;
        if (b < n) {
            const uint32_t have = (uint32_t)min((int64_t)max(d.n_blocks[b], 0), (int64_t)d.max_blocks);
            const uint32_t held = (uint32_t)min(blocks_for(d, d.seq_len[b], d.new_len[b]), (u64)have);
            back = have - held;
            sc.held[b] = held;
        }
        const u64 before = released + sum_before<kWaves>(back, all, share);
        if (b < n)
            sc.released[b] = (uint32_t)before;
        released += all;
    }
    const uint32_t available = (uint32_t)min((u64)free_before + released, (u64)capacity);
    for (uint32_t base = 0; base < n; base += kThreads) {
        const uint32_t b = base + threadIdx.x;
        u64 need = 0, count = 0;
        uint32_t held = 0;
        int32_t status = MAKO_BLOCKS_OK;
        if (b < n) {
            const u64 want = blocks_for(d, d.seq_len[b], d.new_len[b]);
            held = sc.held[b];
            if (want == kWide) {
                status = MAKO_BLOCKS_WIDE;
            } else if (want != kNone) {
                count = (u64)d.new_len[b];
                need = want > held ? want - held : 0;
            }
        }
        const u64 asked_here = asked + sum_before<kWaves>(need, all, share) + need;
        asked += all;
        if (need && asked_here > available)
            status = MAKO_BLOCKS_SHORT;
        if (status)
            count = 0;
        const u64 fit = fitted + sum_before<kWaves>(count, all, share) + count;
        fitted += all;
        if (count && fit > d.max_tokens)
            status = MAKO_BLOCKS_TOKENS;
        if (status)
            need = count = 0;
        const u64 first = tokens + sum_before<kWaves>(count, all, share);
        tokens += all;
        const u64 block = taken + sum_before<kWaves>(need, all, share);
        taken += all;
        if (b < n) {
            d.out_start[b] = (int32_t)first;
            d.out_status[b] = status;
            d.out_n_blocks[b] = (int32_t)(held + need);
            sc.taken[b] = (uint32_t)block;
        }
    }
    if (threadIdx.x == 0) {
        d.out_start[n] = (int32_t)tokens;
        sc.released[n] = (uint32_t)released;
        sc.taken[n] = (uint32_t)taken;
        sc.free_state[0] = free_before;
        sc.free_state[1] = available;
        *d.out_n_free = (int32_t)(available - taken);
    }
}

// The request that entry e is of, by the running sums' n + 1 entries: the last one that begins at or before it.
template <class T>
__device__ __forceinline__ uint32_t owner(const T* sums, uint32_t n, uint32_t e)
{
    uint32_t low = 0, high = n; // sums[low] <= e < sums[high]
    while (high - low > 1) {
        const uint32_t mid = (low + high) / 2;
        if ((uint32_t)sums[mid] <= e)
            low = mid;
        else
            high = mid;
    }
    return low;
}

__global__ void __launch_bounds__(256) apply_kernel(mako_blocks_desc d, Scratch sc)
{
    const uint32_t n = d.n_requests, tokens = (uint32_t)d.out_start[n], taken = sc.taken[n];
    const uint32_t free_before = sc.free_state[0], available = sc.free_state[1];
    const uint32_t step = gridDim.x * 256u, from = blockIdx.x * 256u + threadIdx.x;
    // entry e of those that are given back in this call: where it stands in its table (nothing is written there)
    auto given = [&](uint32_t e) {
        const uint32_t b = owner(sc.released, n, e);
        return d.block_table[(int64_t)b * d.table_stride + sc.held[b] + (e - sc.released[b])];
    };
    // the k-th block that is taken: from the top of the list down, what has just been given back first
    auto get = [&](uint32_t k) {
        const uint32_t at = available - 1u - k;
        return at < free_before ? d.free_blocks[at] : given(at - free_before);
    };
    for (uint32_t e = from; e < available - free_before; e += step)
        d.free_blocks[free_before + e] = given(e);
    for (uint32_t k = from; k < taken; k += step) {
        const uint32_t b = owner(sc.taken, n, k);
        d.block_table[(int64_t)b * d.table_stride + sc.held[b] + (k - sc.taken[b])] = get(k);
    }
    for (uint32_t t = from; t < d.max_tokens; t += step) {
        int64_t slot = -1;
        uint32_t position = 0;
        int32_t request = -1;
        if (t < tokens) {
            const uint32_t b = owner(d.out_start, n, t);
            request = (int32_t)b;
            position = (uint32_t)d.seq_len[b] + (t - (uint32_t)d.out_start[b]);
            const uint32_t at = position / d.block_size, held = sc.held[b];
            // (a block that this call puts into the table is looked up where it comes from)
            const int32_t block = at < held ? d.block_table[(int64_t)b * d.table_stride + at] : get(sc.taken[b] + (at - held));
            slot = (int64_t)block * d.block_size + position % d.block_size;
        }
        d.out_slots[t] = slot;
        if (d.out_positions)
            d.out_positions[t] = (int32_t)position;
        if (d.out_request)
            d.out_request[t] = request;
    }
}

} // namespace

void launch_blocks(hipStream_t st, const mako_blocks_desc& d, const Scratch& sc)
{
    hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(kThreads), 0, st, d, sc);
    const uint32_t items = max(d.max_tokens, d.n_requests);
    hipLaunchKernelGGL(apply_kernel, dim3(min((items + 255u) / 256u, 2048u)), dim3(256), 0, st, d, sc);
}

} // namespace step
} // namespace mako
