// Rows' cuts: what temperature, min_p, top_k and top_p leave of a row of logits (mako_step_cut_rows).
//
//   chunk_kernel  every chunk of 1024 logits, a wave each: its largest logit, its tokens' number, its weights' sum
//   row_kernel    every row, a workgroup each: the chunks together; a row that is cut is read again, for a histogram and
//                 for the tokens around the cut
//   probs_kernel  where asked for: the rows as probabilities
#include "step_common.h"
#include "step_launch.h"

namespace mako {
namespace step {
namespace {

template <class E>
__global__ void __launch_bounds__(256) chunk_kernel(mako_cut_desc d, Scratch sc)
{
    const uint32_t row = blockIdx.y, chunk = blockIdx.x * 4u + (uint32_t)wave(), begin = chunk * kChunk;
    if (begin >= d.n_vocab)
        return;
    const float temperature = d.params[row / d.rows_per_params].temperature;
    const void* x_row = static_cast<const typename E::raw*>(d.logits) + (int64_t)row * d.logits_stride;
    const uint32_t* mask = d.mask ? d.mask + (int64_t)row * d.mask_stride : nullptr;
    float x[16];
#pragma unroll
    for (uint32_t j = 0; j < 16u / E::kVec; ++j)
        load_tokens<E>(x_row, mask, begin + (j * 64u + (uint32_t)lane()) * E::kVec, d.n_vocab, x + j * E::kVec);
    float m = x[0];
    uint32_t count = 0;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        m = fmaxf(m, x[k]);
        count += (uint32_t)__popcll(__ballot(x[k] > -INFINITY));
    }
    m = __ockl_wfred_max_f32(m);
    double sum = 0.0;
    if (temperature > 0.0f && count) {
        const double scale = weight_scale(temperature), md = (double)m;
#pragma unroll
        for (int k = 0; k < 16; ++k)
            sum += weight(x[k], md, scale);
        sum = __ockl_wfred_add_f64(sum);
    }
    if (lane() == 0)
        sc.chunks[(uint64_t)row * sc.chunks_cap + chunk] = {sum, m, count};
}

constexpr int kRowThreads = 1024, kRowWaves = kRowThreads / 64;
constexpr uint32_t kBins = 2048;
constexpr uint32_t kList = 8192; // tokens around a cut that are put in order in LDS

struct RowLds {
    uint64_t list[kList];
    uint64_t bin_mass[kBins]; // weights in units of 2^-unit
    uint64_t digit_mass[kBins];
    uint32_t bin_count[kBins];
    uint32_t digit_count[kBins];
    Share<kRowWaves> share;
    uint32_t n, at, id;
    double mass;
    uint64_t u0, u1, u2;
};

// What the passes over a row need to know of it.
template <class E>
struct Row {
    const void* x;
    const uint32_t* mask;
    uint32_t n;
    float max;
    double scale;    // of weights
    float bin_scale; // of bins: bin(x) = (max - x) bin_scale, a function that never falls as x does
    int unit;        // weights are added up as whole multiples of 2^-unit, in any order

    __device__ __forceinline__ uint32_t bin(float v) const
    {
        return (uint32_t)fminf((max - v) * bin_scale, (float)(kBins - 1u));
    }
    __device__ __forceinline__ double weigh(float v) const { return weight(v, (double)max, scale); }
    __device__ __forceinline__ uint64_t units(double w) const { return (uint64_t)ldexp(w, unit); }
    __device__ __forceinline__ double mass(uint64_t u) const { return ldexp((double)u, -unit); }

    // f(token, logit) for every token of the row
    template <class F>
    __device__ __forceinline__ void each(F f) const
    {
        constexpr uint32_t kStep = kRowThreads * E::kVec, kAhead = 2;
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

// The first of kBins bins (two to a thread) with which the running count or mass gets where the cut is: its number in
// lds.at, what lies before it in lds.u0 (count) and lds.u1 (mass units), its own count in lds.n.
template <class E>
__device__ void find_bin(const Row<E>& row, const uint32_t* count, const uint64_t* mass, const Want& want, uint64_t count0, uint64_t mass0, RowLds& lds)
{
    const uint32_t a = 2u * threadIdx.x;
    const unsigned long long c[2] = {count[a], count[a + 1]}, m[2] = {mass[a], mass[a + 1]};
    unsigned long long all;
    unsigned long long cb = count0 + sum_before<kRowWaves>(c[0] + c[1], all, lds.share);
    unsigned long long mb = mass0 + sum_before<kRowWaves>(m[0] + m[1], all, lds.share);
    // (the last bin with a token, should no bin get there)
    const uint32_t last = ~all_min<kRowWaves>(~(c[1] ? a + 2u : (c[0] ? a + 1u : 0u)), lds.share);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const bool there = c[k] != 0 && (want.by_rank ? cb + c[k] >= want.rank : row.mass(mb + m[k]) >= want.mass);
        const bool sooner = want.by_rank ? cb >= want.rank : (cb != 0 && row.mass(mb) >= want.mass);
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
    for (uint32_t i = n + threadIdx.x; i < size; i += kRowThreads)
        list[i] = ~0ull;
    __syncthreads();
    for (uint32_t k = 2; k <= size; k *= 2)
        for (uint32_t j = k / 2; j; j /= 2) {
            for (uint32_t t = threadIdx.x; t < size / 2; t += kRowThreads) {
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

// The cut of a row whose bins are filled.
template <class E>
__device__ Cut find_cut(const Row<E>& row, const Want& want, RowLds& lds)
{
    find_bin(row, lds.bin_count, lds.bin_mass, want, 0, 0, lds);
    const uint32_t bin = lds.at;
    uint64_t before = lds.u0, mass_before = lds.u1;
    uint32_t count = lds.n;
    __syncthreads();
    // a crowded bin is divided by its tokens' order keys, digit by digit from the top, until few enough are left
    uint32_t shift = 32, prefix = 0;
    auto in = [&](float v) { return row.bin(v) == bin && (shift == 32u || order_key(v) >> shift == prefix); };
    while (count > kList && shift) {
        const uint32_t bits = shift == 10u ? 10u : 11u, next = shift - bits;
        for (uint32_t i = threadIdx.x; i < kBins; i += kRowThreads) {
            lds.digit_count[i] = 0;
            lds.digit_mass[i] = 0;
        }
        __syncthreads();
        row.each([&](uint32_t, float v) {
            if (in(v)) {
                const uint32_t digit = (order_key(v) >> next) & ((1u << bits) - 1u);
                atomicAdd(&lds.digit_count[digit], 1u);
                atomicAdd((unsigned long long*)&lds.digit_mass[digit], (unsigned long long)row.units(row.weigh(v)));
            }
        });
        __syncthreads();
        find_bin(row, lds.digit_count, lds.digit_mass, want, before, mass_before, lds);
        prefix = (shift == 32u ? 0u : prefix << bits) | lds.at;
        before = lds.u0;
        mass_before = lds.u1;
        count = lds.n;
        shift = next;
        __syncthreads();
    }
    Cut cut;
    if (count > kList) {
        // nothing but equal logits: the cut is behind so many of them, in the tokens' order
        const float v = key_logit(prefix);
        const double w = row.weigh(v);
        uint32_t rank = want.by_rank ? want.rank - (uint32_t)before : 0u;
        if (!want.by_rank) {
            const double r = ceil((want.mass - row.mass(mass_before)) / w);
            rank = r >= (double)count ? count : (r < 1.0 ? 1u : (uint32_t)r);
        }
        uint32_t seen = 0;
        constexpr uint32_t kStep = kRowThreads * E::kVec;
        for (uint32_t base = 0; base < row.n; base += kStep) {
            float x[E::kVec];
            load_tokens<E>(row.x, row.mask, base + threadIdx.x * E::kVec, row.n, x);
            uint32_t mine = 0;
#pragma unroll
            for (uint32_t k = 0; k < E::kVec; ++k)
                mine += x[k] == v;
            unsigned long long all;
            uint32_t at = seen + (uint32_t)sum_before<kRowWaves>((unsigned long long)mine, all, lds.share);
#pragma unroll
            for (uint32_t k = 0; k < E::kVec; ++k)
                if (x[k] == v && ++at == rank)
                    lds.id = base + threadIdx.x * E::kVec + k;
            seen += (uint32_t)all;
            if (seen >= rank)
                break;
        }
        __syncthreads();
        cut = {(uint32_t)before + rank, row.mass(mass_before) + (double)rank * w, v, lds.id};
        __syncthreads();
        return cut;
    }
    if (threadIdx.x == 0)
        lds.n = 0;
    __syncthreads();
    row.each([&](uint32_t id, float v) {
        if (in(v)) {
            const uint32_t at = atomicAdd(&lds.n, 1u);
            if (at < kList) // (always: `count` of them)
                lds.list[at] = (uint64_t)order_key(v) << 32 | id;
        }
    });
    __syncthreads();
    sort_list(lds.list, count);
    // (a stretch of the list to each thread)
    const uint32_t each = (count + kRowThreads - 1) / kRowThreads, from = min(threadIdx.x * each, count), to = min(from + each, count);
    double mine = 0.0, all;
    for (uint32_t i = from; i < to; ++i)
        mine += row.weigh(key_logit((uint32_t)(lds.list[i] >> 32)));
    double sum = sum_before<kRowWaves>(mine, all, lds.share);
    const double base = row.mass(mass_before);
    uint32_t here = kNoToken;
    double here_mass = 0.0;
    for (uint32_t i = from; i < to; ++i) {
        sum += row.weigh(key_logit((uint32_t)(lds.list[i] >> 32)));
        if (here == kNoToken && (i + 1 == count || (want.by_rank ? before + i + 1 >= want.rank : base + sum >= want.mass))) {
            here = i;
            here_mass = base + sum;
        }
    }
    const uint32_t first = all_min<kRowWaves>(here, lds.share);
    if (here == first)
        lds.mass = here_mass;
    __syncthreads();
    const uint64_t last = lds.list[first];
    cut = {(uint32_t)before + first + 1u, lds.mass, key_logit((uint32_t)(last >> 32)), (uint32_t)last};
    __syncthreads();
    return cut;
}

template <class E>
__global__ void __launch_bounds__(kRowThreads) row_kernel(mako_cut_desc d, Scratch sc)
{
    extern __shared__ unsigned char dyn[];
    RowLds& lds = *reinterpret_cast<RowLds*>(dyn);
    const uint32_t r = blockIdx.x;
    const mako_sampling_params p = d.params[r / d.rows_per_params];
    const bool greedy = !(p.temperature > 0.0f);
    Row<E> row;
    row.x = static_cast<const typename E::raw*>(d.logits) + (int64_t)r * d.logits_stride;
    row.mask = d.mask ? d.mask + (int64_t)r * d.mask_stride : nullptr;
    row.n = d.n_vocab;
    row.scale = weight_scale(p.temperature);
    const uint32_t chunks = (d.n_vocab + kChunk - 1) / kChunk;
    ChunkRec rec = {0.0, -INFINITY, 0};
    if (threadIdx.x < chunks)
        rec = sc.chunks[(uint64_t)r * sc.chunks_cap + threadIdx.x];
    row.max = all_max<kRowWaves>(rec.max, lds.share);
    const uint32_t count = all_sum<kRowWaves>(rec.count, lds.share);
    mako_row_cut out;
    out.max_logit = row.max;
    out.temperature = greedy ? 0.0f : p.temperature;
    out.cut_logit = -INFINITY;
    out.cut_token = -1;
    out.n_kept = count;
    out.total = 0.0;
    out.top_token = -1;
    if (count) {
        // the first token: in the first chunk that has the largest logit
        const uint32_t chunk = all_min<kRowWaves>(rec.count && rec.max == row.max ? threadIdx.x : kNoToken, lds.share);
        const uint32_t i = chunk * kChunk + threadIdx.x;
        uint32_t id = kNoToken;
        if (i < d.n_vocab) {
            const typename E::raw v = static_cast<const typename E::raw*>(row.x)[i];
            if (token_logit(E::of(v, 0), !row.mask || (row.mask[i >> 5] >> (i & 31u) & 1u)) == row.max)
                id = i;
        }
        out.top_token = (int32_t)all_min<kRowWaves>(id, lds.share);
        if (greedy) {
            out.total = 1.0;
            if (count > 1) {
                out.n_kept = 1;
                out.cut_logit = row.max;
                out.cut_token = out.top_token;
            }
        } else {
            out.total = all_sum<kRowWaves>(rec.count ? rec.sum * weight(rec.max, (double)row.max, row.scale) : 0.0, lds.share);
            const bool min_p = p.min_p > 0.0f, top_p = p.top_p < 1.0f;
            if (min_p || top_p || (p.top_k && p.top_k < count)) {
                // bins over four times what lies between the largest logit and the one of the mean weight
                const double gap = log((double)count / out.total) * kLog2e / row.scale;
                row.bin_scale = (float)fmin((double)kBins / fmax(4.0 * gap, 1e-30), 1e30);
                row.unit = 60 - ilogb(out.total);
                for (uint32_t i = threadIdx.x; i < kBins; i += kRowThreads) {
                    lds.bin_count[i] = 0;
                    lds.bin_mass[i] = 0;
                }
                __syncthreads();
                uint32_t above = 0;
                row.each([&](uint32_t, float v) {
                    const uint32_t b = row.bin(v);
                    const double w = row.weigh(v);
                    above += w >= (double)p.min_p;
                    atomicAdd(&lds.bin_count[b], 1u);
                    atomicAdd((unsigned long long*)&lds.bin_mass[b], (unsigned long long)row.units(w));
                });
                uint32_t rank = count;
                if (min_p)
                    rank = max(all_sum<kRowWaves>(above, lds.share), 1u);
                if (p.top_k)
                    rank = min(rank, p.top_k);
                __syncthreads();
                Cut cut = {count, out.total, 0.0f, 0};
                if (rank < count)
                    cut = find_cut(row, Want{true, rank, 0.0}, lds);
                if (top_p)
                    cut = find_cut(row, Want{false, 0, (double)p.top_p * cut.mass}, lds);
                if (cut.n < count) {
                    out.total = cut.mass;
                    out.n_kept = cut.n;
                    out.cut_logit = cut.x;
                    out.cut_token = (int32_t)cut.id;
                }
            }
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
        const uint32_t i = blockIdx.x * kSlice + (j * 256u + threadIdx.x) * E::kVec;
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
    hipLaunchKernelGGL(chunk_kernel<E>, dim3((d.n_vocab + kSlice - 1) / kSlice, d.n_rows), dim3(256), 0, st, d, sc);
    hipLaunchKernelGGL(row_kernel<E>, dim3(d.n_rows), dim3(kRowThreads), sizeof(RowLds), st, d, sc);
}
template <class E>
void probs(hipStream_t st, const mako_cut_desc& d)
{
    hipLaunchKernelGGL(probs_kernel<E>, dim3((d.n_vocab + kSlice - 1) / kSlice, d.n_rows), dim3(256), 0, st, d);
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
    d.logits_type == MAKO_LOGITS_F32 ? cut<F32>(st, d, sc) : (d.logits_type == MAKO_LOGITS_BF16 ? cut<BF16>(st, d, sc) : cut<F16>(st, d, sc));
}

void launch_probs(hipStream_t st, const mako_cut_desc& d)
{
    d.logits_type == MAKO_LOGITS_F32 ? probs<F32>(st, d) : (d.logits_type == MAKO_LOGITS_BF16 ? probs<BF16>(st, d) : probs<F16>(st, d));
}

} // namespace step
} // namespace mako
