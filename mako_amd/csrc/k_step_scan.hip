// The passes over the rows of mako_step_cut_rows: a wave for every chunk of a row, with no word between waves.
//   scan_kernel  every row
//   look_kernel  the rows that have a plan: the tokens around the cut, and what lies above them or below
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

// A chunk's logits, 16 to a lane; -inf: no token.
template <class E>
struct Chunk {
    uint32_t begin;
    float x[16];

    // (the k-th logit's token)
    __device__ __forceinline__ uint32_t token(int k) const { return begin + ((uint32_t)k / E::kVec * 64u + (uint32_t)lane()) * E::kVec + (uint32_t)k % E::kVec; }

    __device__ __forceinline__ Chunk(const mako_cut_desc& d, uint32_t row, uint32_t chunk) : begin(chunk * kChunk)
    {
        const void* x_row = static_cast<const typename E::raw*>(d.logits) + (int64_t)row * d.logits_stride;
        const uint32_t* mask = d.mask ? d.mask + (int64_t)row * d.mask_stride : nullptr;
#pragma unroll
        for (int k = 0; k < 16; k += (int)E::kVec)
            load_vec<E>(x_row, token(k), d.n_vocab, x + k);
#pragma unroll
        for (int k = 0; k < 16; ++k)
            x[k] = fmaxf(x[k], -INFINITY); // (of a NaN and a number, the number)
        if (mask) {
#pragma unroll
            for (int k = 0; k < 16; k += (int)E::kVec) {
                const uint32_t i = token(k), bits = i < d.n_vocab ? mask[i >> 5] >> (i & 31u) : 0u;
#pragma unroll
                for (int e = 0; e < (int)E::kVec; ++e)
                    if (!((bits >> e) & 1u))
                        x[k + e] = -INFINITY;
            }
        }
    }
    __device__ __forceinline__ void no_infinity()
    {
#pragma unroll
        for (int k = 0; k < 16; ++k)
            x[k] = fminf(x[k], kFltMax);
    }
    // The tokens of `in` (a bit for every lane's k-th) into a list.
    __device__ __forceinline__ void list(const unsigned long long* in, uint64_t* to) const
    {
        const unsigned long long before = (1ull << lane()) - 1ull;
        uint32_t base = 0;
#pragma unroll
        for (int k = 0; k < 16; ++k)
            if (in[k]) {
                if (in[k] >> lane() & 1ull)
                    to[base + (uint32_t)__popcll(in[k] & before)] = (uint64_t)order_key(x[k] + 0.0f) << 32 | token(k);
                base += (uint32_t)__popcll(in[k]);
            }
    }
};

template <class E>
__global__ void __launch_bounds__(256, 8) scan_kernel(mako_cut_desc d, Scratch sc)
{
    const uint32_t row = blockIdx.y, chunk = blockIdx.x * 4u + (uint32_t)wave(), chunks = chunks_of(d.n_vocab);
    if (row == 0 && chunk == 0 && lane() == 0)
        sc.wide[0] = 0;
    if (chunk >= chunks)
        return;
    Chunk<E> c(d, row, chunk);
    float(&x)[16] = c.x;
    const RowKind kind(d.params[row / d.rows_per_params]);
    float mine = -INFINITY;
    ChunkRec rec = {0.0, -INFINITY, -INFINITY, 0u, 0u, kNoToken, INFINITY};
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        mine = fmaxf(mine, x[k]);
        rec.count += (uint32_t)__popcll(__ballot(x[k] > -INFINITY));
    }
    rec.max = __ockl_wfred_max_f32(mine);
    if (rec.max == INFINITY) {
        c.no_infinity();
        mine = fminf(mine, kFltMax);
        rec.max = kFltMax;
    }
    const uint64_t at = (uint64_t)row * sc.chunks_cap + chunk;
    if (rec.count) {
        uint32_t id = kNoToken;
        if (mine == rec.max) {
#pragma unroll
            for (int k = 15; k >= 0; --k)
                id = x[k] == rec.max ? c.token(k) : id;
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
                c.list(in, sc.lists + at * kChunkList);
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
__global__ void __launch_bounds__(256, 6) look_kernel(mako_cut_desc d, Scratch sc)
{
    __shared__ float weighed[4][kChunk];
    const uint32_t chunks = chunks_of(d.n_vocab), groups = (chunks + 3) / 4, items = sc.wide[0] * groups;
    for (uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
        const uint32_t row = sc.wide[1 + item / groups], chunk = item % groups * 4u + (uint32_t)wave();
        const RowPlan& plan = sc.plans[row];
        if (!plan.look || chunk >= chunks)
            continue;
        const float low = plan.low, high = plan.high;
        const bool from_above = plan.from_above;
        const float max = d.out_cuts[row].max_logit;
        const double scale = weight_scale(d.out_cuts[row].temperature);
        Chunk<E> c(d, row, chunk);
        if (max == kFltMax)
            c.no_infinity();
        ChunkRec rec = {0.0, 0.0f, 0.0f, 0u, 0u, 0u, 0.0f};
        unsigned long long in[16];
        const unsigned long long before = (1ull << lane()) - 1ull;
        // (what is weighed moves together first: where it is one logit in ten, nearly every 64 have one)
        float* const mine = weighed[wave()];
        uint32_t n = 0;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const float x = c.x[k];
            const unsigned long long up = __ballot(x >= high);
            in[k] = __ballot(x >= low) & ~up;
            rec.count += (uint32_t)__popcll(up);
            rec.n_list += (uint32_t)__popcll(in[k]);
            const unsigned long long side = from_above ? up : __ballot(x > -INFINITY) & ~(up | in[k]);
            if (side) {
                if (side >> lane() & 1ull)
                    mine[n + (uint32_t)__popcll(side & before)] = x;
                n += (uint32_t)__popcll(side);
            }
        }
        const uint64_t at = (uint64_t)row * sc.chunks_cap + chunk;
        if (rec.n_list <= kChunkList)
            c.list(in, sc.lists + at * kChunkList);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        double sum = 0.0;
        for (uint32_t i = (uint32_t)lane(); i < n; i += 64u)
            sum += weight(mine[i], (double)max, scale);
        __builtin_amdgcn_wave_barrier();
        rec.sum = __ockl_wfred_add_f64(sum);
        if (lane() == 0)
            sc.chunks[at] = rec;
    }
}

template <class E>
void scan(hipStream_t st, const mako_cut_desc& d, const Scratch& sc)
{
    hipLaunchKernelGGL(scan_kernel<E>, dim3((chunks_of(d.n_vocab) + 3) / 4, d.n_rows), dim3(256), 0, st, d, sc);
}

constexpr uint32_t kLookWorkgroups = 4096;
template <class E>
void look(hipStream_t st, const mako_cut_desc& d, const Scratch& sc)
{
    const uint32_t items = d.n_rows * ((chunks_of(d.n_vocab) + 3) / 4); // (65535 rows of 256 at most)
    hipLaunchKernelGGL(look_kernel<E>, dim3(items < kLookWorkgroups ? items : kLookWorkgroups), dim3(256), 0, st, d, sc);
}

} // namespace

void launch_scan(hipStream_t st, const mako_cut_desc& d, const Scratch& sc)
{
    d.logits_type == MAKO_LOGITS_F32 ? scan<F32>(st, d, sc) : (d.logits_type == MAKO_LOGITS_BF16 ? scan<BF16>(st, d, sc) : scan<F16>(st, d, sc));
}

void launch_look(hipStream_t st, const mako_cut_desc& d, const Scratch& sc)
{
    d.logits_type == MAKO_LOGITS_F32 ? look<F32>(st, d, sc) : (d.logits_type == MAKO_LOGITS_BF16 ? look<BF16>(st, d, sc) : look<F16>(st, d, sc));
}

} // namespace step
} // namespace mako
