// The pass over the rows of mako_step_cut_rows: a wave for every chunk of every row, with no word between waves.
#include "step_common.h"
#include "step_cut.h"
#include "step_launch.h"

namespace mako {
namespace step {
namespace {

// A lower bound of the n-th largest of the wave's values (of the least, if fewer lanes have a token; one has), to 16 bits of
// their order.
__device__ __forceinline__ float nth_largest(float v, uint32_t n)
{
    n = min(n, (uint32_t)__popcll(__ballot(v > -INFINITY)));
    const uint32_t key = ~order_key(v); // (rises with v)
    uint32_t found = 0;
#pragma unroll
    for (int bit = 31; bit >= 16; --bit) {
        const uint32_t trial = found | 1u << bit;
        if ((uint32_t)__popcll(__ballot(key >= trial)) >= n)
            found = trial;
    }
    return key_logit(~found);
}

template <class E>
__global__ void __launch_bounds__(256, 8) scan_kernel(mako_cut_desc d, Scratch sc)
{
    const uint32_t row = blockIdx.y, chunk = blockIdx.x * 4u + (uint32_t)wave(), begin = chunk * kChunk, chunks = chunks_of(d.n_vocab);
    if (chunk >= chunks)
        return;
    const void* x_row = static_cast<const typename E::raw*>(d.logits) + (int64_t)row * d.logits_stride;
    const uint32_t* mask = d.mask ? d.mask + (int64_t)row * d.mask_stride : nullptr;
    // (a lane's k-th logit)
    auto place = [&](int k) { return begin + ((uint32_t)k / E::kVec * 64u + (uint32_t)lane()) * E::kVec + (uint32_t)k % E::kVec; };
    float x[16]; // (-inf: no token)
#pragma unroll
    for (int k = 0; k < 16; k += (int)E::kVec)
        load_vec<E>(x_row, place(k), d.n_vocab, x + k);
    const RowKind kind(d.params[row / d.rows_per_params]);
#pragma unroll
    for (int k = 0; k < 16; ++k)
        x[k] = fmaxf(x[k], -INFINITY); // (of a NaN and a number, the number)
    if (mask) {
#pragma unroll
        for (int k = 0; k < 16; k += (int)E::kVec) {
            const uint32_t i = place(k), bits = i < d.n_vocab ? mask[i >> 5] >> (i & 31u) : 0u;
#pragma unroll
            for (int e = 0; e < (int)E::kVec; ++e)
                if (!((bits >> e) & 1u))
                    x[k + e] = -INFINITY;
        }
    }
    float mine = -INFINITY;
    ChunkRec rec = {0.0, -INFINITY, -INFINITY, 0u, 0u, kNoToken, INFINITY};
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        mine = fmaxf(mine, x[k]);
        rec.count += (uint32_t)__popcll(__ballot(x[k] > -INFINITY));
    }
    rec.max = __ockl_wfred_max_f32(mine);
    if (rec.max == INFINITY) {
#pragma unroll
        for (int k = 0; k < 16; ++k)
            x[k] = fminf(x[k], kFltMax);
        mine = fminf(mine, kFltMax);
        rec.max = kFltMax;
    }
    const uint64_t at = (uint64_t)row * sc.chunks_cap + chunk;
    if (rec.count) {
        uint32_t id = kNoToken;
        if (mine == rec.max) {
#pragma unroll
            for (int k = 15; k >= 0; --k)
                id = x[k] == rec.max ? place(k) : id;
        }
        rec.first = __ockl_wfred_min_u32(id);
        if (kind.sums) {
            const double md = (double)rec.max;
            // (weights below 2^-64 of the largest are nothing beside it)
            if (rec.count > 1) {
                double sum = 0.0;
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    sum += weight(x[k], md, kind.scale);
                rec.sum = __ockl_wfred_add_f64(sum);
            } else {
                rec.sum = 1.0;
            }
        }
        if (kind.min_p) {
            float low = INFINITY;
#pragma unroll
            for (int k = 0; k < 16; ++k)
                low = fminf(low, x[k] > -INFINITY ? x[k] : INFINITY);
            rec.low = -__ockl_wfred_max_f32(-low);
        }
        if (kind.cut) {
            // the chunk's first tokens: those not below the n-th largest of the lanes' largest; above it, where these are too
            // many (equal ones); none, where these are too many too.  A chunk of few tokens lists them all.
            rec.listed = nth_largest(mine, kind.list_length(chunks));
            unsigned long long in[16];
            auto take = [&](bool above) {
                rec.n_list = 0;
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    in[k] = __ballot(above ? x[k] > rec.listed : x[k] >= rec.listed);
                    rec.n_list += (uint32_t)__popcll(in[k]);
                }
            };
            if (rec.count <= kChunkList)
                rec.listed = -kFltMax;
            take(false);
            bool strict = false;
            if (rec.n_list > kChunkList) {
                take(true);
                strict = true;
            }
            if (rec.n_list > kChunkList) {
                rec.n_list = 0;
                rec.listed = INFINITY;
            } else {
                uint64_t* list = sc.lists + at * kChunkList;
                const unsigned long long before = (1ull << lane()) - 1ull;
                uint32_t base = 0;
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    if (in[k]) {
                        if (in[k] >> lane() & 1ull)
                            list[base + (uint32_t)__popcll(in[k] & before)] = (uint64_t)order_key(x[k] + 0.0f) << 32 | place(k);
                        base += (uint32_t)__popcll(in[k]);
                    }
                }
                if (strict) // (the next larger number)
                    rec.listed = key_logit(order_key(rec.listed + 0.0f) - 1u);
                if (rec.count <= kChunkList)
                    rec.listed = -INFINITY;
            }
        }
    }
    rec.max += 0.0f;
    if (lane() == 0)
        sc.chunks[at] = rec;
}

template <class E>
void scan(hipStream_t st, const mako_cut_desc& d, const Scratch& sc)
{
    hipLaunchKernelGGL(scan_kernel<E>, dim3((chunks_of(d.n_vocab) + 3) / 4, d.n_rows), dim3(256), 0, st, d, sc);
}

} // namespace

void launch_scan(hipStream_t st, const mako_cut_desc& d, const Scratch& sc)
{
    d.logits_type == MAKO_LOGITS_F32 ? scan<F32>(st, d, sc) : (d.logits_type == MAKO_LOGITS_BF16 ? scan<BF16>(st, d, sc) : scan<F16>(st, d, sc));
}

} // namespace step
} // namespace mako
