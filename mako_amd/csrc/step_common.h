// What the kernels of a speculative decode step share: rows of logits of three types, weights in 64 bits, the order of a
// row's tokens, and a workgroup's reductions and scans.  (The entry points: mako_step.hip.)
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/mako_step.h"

extern "C" __device__ uint32_t __ockl_wfred_add_u32(uint32_t);
extern "C" __device__ uint32_t __ockl_wfred_min_u32(uint32_t);
extern "C" __device__ uint32_t __ockl_wfred_max_u32(uint32_t);
extern "C" __device__ float __ockl_wfred_max_f32(float);
extern "C" __device__ double __ockl_wfred_add_f64(double);
extern "C" __device__ uint32_t __ockl_wfscan_add_u32(uint32_t, bool inclusive);
extern "C" __device__ double __ockl_wfscan_add_f64(double, bool inclusive);
extern "C" __device__ uint64_t __ockl_wfscan_add_u64(uint64_t, bool inclusive);

namespace mako {
namespace step {

constexpr uint32_t kPart = 1024;        // logits of a row that a workgroup of 256 threads takes: 4 a thread
constexpr uint32_t kNoToken = 0xffffffffu;
constexpr float kFltMax = 3.402823466e+38f;
constexpr double kLog2e = 1.4426950408889634;

// ---- types of logits: kVec of them are the 16 bytes that a lane loads at once ----
// (a row may begin at any element: the loads promise no more than that)
typedef uint32_t words_at_4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t words_at_2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t pair_at_2 __attribute__((ext_vector_type(2), aligned(2)));
struct F32 {
    using raw = uint32_t;
    using words = words_at_4;
    static constexpr uint32_t kVec = 4;
    static __device__ __forceinline__ float of(uint32_t w, int) { return __uint_as_float(w); }
};
struct BF16 {
    using raw = uint16_t;
    using words = words_at_2;
    static constexpr uint32_t kVec = 8;
    static __device__ __forceinline__ float of(uint32_t w, int k) { return __uint_as_float(k & 1 ? w & 0xffff0000u : w << 16); }
};
struct F16 {
    using raw = uint16_t;
    using words = words_at_2;
    static constexpr uint32_t kVec = 8;
    static __device__ __forceinline__ float of(uint32_t w, int k)
    {
        return (float)__builtin_bit_cast(_Float16, (uint16_t)(k & 1 ? w >> 16 : w));
    }
};

// Logits i .. i + kVec - 1 of a row, as fp32.
template <class E>
__device__ __forceinline__ void load_whole(const void* row, uint32_t i, float* x)
{
    using raw = typename E::raw;
    const typename E::words w = *reinterpret_cast<const typename E::words*>(static_cast<const raw*>(row) + i);
#pragma unroll
    for (uint32_t k = 0; k < E::kVec; ++k)
        x[k] = E::of(sizeof(raw) == 4 ? w[k % 4] : w[k / 2], (int)k);
}
// ... of a row of n; those at n and behind are NaN (no token).
template <class E>
__device__ __forceinline__ void load_vec(const void* row, uint32_t i, uint32_t n, float* x)
{
    if (i + E::kVec <= n) {
        load_whole<E>(row, i, x);
    } else {
#pragma unroll
        for (uint32_t k = 0; k < E::kVec; ++k) {
            x[k] = __uint_as_float(0x7fc00000u);
            if (i + k < n)
                x[k] = E::of(static_cast<const typename E::raw*>(row)[i + k], 0);
        }
    }
}

// Four logits from i on (a multiple of four), the same way.
template <class E>
__device__ __forceinline__ void load_whole_four(const void* row, uint32_t i, float* x)
{
    if (sizeof(typename E::raw) == 4) {
        load_whole<E>(row, i, x);
    } else {
        const pair_at_2 w = *reinterpret_cast<const pair_at_2*>(static_cast<const typename E::raw*>(row) + i);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            x[k] = E::of(w[k / 2], k);
    }
}
template <class E>
__device__ __forceinline__ void load_four(const void* row, uint32_t i, uint32_t n, float* x)
{
    if (i + 4u <= n) {
        load_whole_four<E>(row, i, x);
    } else {
#pragma unroll
        for (uint32_t k = 0; k < 4u; ++k) {
            x[k] = __uint_as_float(0x7fc00000u);
            if (i + k < n)
                x[k] = E::of(static_cast<const typename E::raw*>(row)[i + k], 0);
        }
    }
}

// A logit as the operators see it: -inf for what is no token (masked, NaN, -inf), +inf as the largest finite value, and
// -0 as 0 (the two are equal, and are one value to order_key()).
__device__ __forceinline__ float token_logit(float x, bool allowed)
{
    return allowed && x > -INFINITY ? fminf(x, kFltMax) + 0.0f : -INFINITY;
}

// N vectors of a row's logits as token_logit() gives them, the a-th from token at(a) on (a multiple of kVec: its mask bits lie in one
// word), all asked for before any is looked at.
template <class E, uint32_t N, class F>
__device__ __forceinline__ void load_tokens(const void* row, const uint32_t* mask, F at, uint32_t n, float (&x)[N][E::kVec])
{
#pragma unroll
    for (uint32_t a = 0; a < N; ++a)
        load_vec<E>(row, at(a), n, x[a]);
    if (mask) {
        uint32_t bits[N];
#pragma unroll
        for (uint32_t a = 0; a < N; ++a)
            bits[a] = at(a) < n ? mask[at(a) >> 5] >> (at(a) & 31u) : 0u;
#pragma unroll
        for (uint32_t a = 0; a < N; ++a)
#pragma unroll
            for (uint32_t k = 0; k < E::kVec; ++k) {
                const uint32_t keep = (uint32_t)((int32_t)(bits[a] << (31u - k)) >> 31);
                x[a][k] = __uint_as_float((__float_as_uint(x[a][k]) & keep) | (0xff800000u & ~keep));
            }
    }
#pragma unroll
    for (uint32_t a = 0; a < N; ++a)
#pragma unroll
        for (uint32_t k = 0; k < E::kVec; ++k)
            x[a][k] = fminf(fmaxf(x[a][k], -INFINITY), kFltMax) + 0.0f; // (of a NaN and a number, the number)
}

// Rising keys are falling logits.
__device__ __forceinline__ uint32_t order_key(float x)
{
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? u : ~(u | 0x80000000u);
}
__device__ __forceinline__ float key_logit(uint32_t k)
{
    return __uint_as_float(k & 0x80000000u ? k : ~k & 0x7fffffffu);
}

// 2^t for t <= 0: 2^round(t) times a polynomial in the rest, of degree 9: of those with a constant term of 1 the one whose largest
// relative error over [-1/2, 1/2] is least (found by exchange), 1.6e-14 with its roundings (degree 10: 2e-16, and an operation more
// for each logit).  2^0 is exactly 1.  0 below 2^-1074.  kFinite: t is neither NaN nor -infinity.
template <bool kFinite = false>
__device__ __forceinline__ double exp2_down(double t)
{
    if (!kFinite)
        t = fmax(t, -1100.0);
    const double n = rint(t), f = t - n;
    double p = 1.0148340794092651e-07;
    p = fma(p, f, 1.3258335415197215e-06);
    p = fma(p, f, 1.5252990014502824e-05);
    p = fma(p, f, 0.0001540344088440716);
    p = fma(p, f, 0.001333355762547261);
    p = fma(p, f, 0.009618129181163993);
    p = fma(p, f, 0.05550410866841572);
    p = fma(p, f, 0.2402265069572282);
    p = fma(p, f, 0.6931471805598851);
    p = fma(p, f, 1.0);
    return ldexp(p, (int)n);
}

// N at once, step by step: where few waves run, a chain of fp64 operations is waited for, and N of them are no longer than one.
template <int N>
__device__ __forceinline__ void exp2_down(const double* t, double* out)
{
    constexpr double c[10] = {1.0148340794092651e-07, 1.3258335415197215e-06, 1.5252990014502824e-05, 0.0001540344088440716, 0.001333355762547261,
                              0.009618129181163993, 0.05550410866841572, 0.2402265069572282, 0.6931471805598851, 1.0};
    double n[N], f[N], p[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const double low = fmax(t[k], -1100.0);
        n[k] = rint(low);
        f[k] = low - n[k];
        p[k] = c[0];
    }
#pragma unroll
    for (int i = 1; i < 10; ++i)
#pragma unroll
        for (int k = 0; k < N; ++k)
            p[k] = fma(p[k], f[k], c[i]);
#pragma unroll
    for (int k = 0; k < N; ++k)
        out[k] = ldexp(p[k], (int)n[k]);
}

// log2(e) / T, for weights 2^((x - max) scale).  (T infinite: as good as 0, but 0 times an infinity would be no number.)
__device__ __forceinline__ double weight_scale(float temperature)
{
    return temperature > 0.0f ? fmax(kLog2e / (double)temperature, 1e-300) : 1e-300;
}
// (the difference first: it is exactly 0 for the largest logit, whose weight is exactly 1)
template <bool kFinite = false>
__device__ __forceinline__ double weight(float x, double max_logit, double scale)
{
    return exp2_down<kFinite>(((double)x - max_logit) * scale);
}

__device__ __forceinline__ int lane()
{
    return threadIdx.x & 63;
}
__device__ __forceinline__ int wave()
{
    return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
}

// ---- of a workgroup of W waves; every thread gets the result, and `s` may be used again at once ----
template <int W>
struct Share {
    unsigned long long u[W];
    double d[W];
};

template <int W>
__device__ __forceinline__ uint32_t all_sum(uint32_t v, Share<W>& s)
{
    v = __ockl_wfred_add_u32(v);
    if (lane() == 0)
        s.u[wave()] = v;
    __syncthreads();
    uint32_t t = 0;
    for (int w = 0; w < W; ++w)
        t += (uint32_t)s.u[w];
    __syncthreads();
    return t;
}
template <int W>
__device__ __forceinline__ uint32_t all_min(uint32_t v, Share<W>& s)
{
    v = __ockl_wfred_min_u32(v);
    if (lane() == 0)
        s.u[wave()] = v;
    __syncthreads();
    uint32_t t = 0xffffffffu;
    for (int w = 0; w < W; ++w)
        t = min(t, (uint32_t)s.u[w]);
    __syncthreads();
    return t;
}
// (in a fixed order: the lanes of a wave, then the waves)
template <int W>
__device__ __forceinline__ double all_sum(double v, Share<W>& s)
{
    v = __ockl_wfred_add_f64(v);
    if (lane() == 0)
        s.d[wave()] = v;
    __syncthreads();
    double t = 0.0;
    for (int w = 0; w < W; ++w)
        t += s.d[w];
    __syncthreads();
    return t;
}
// What the threads before this one have; `total`: what all have.
template <int W>
__device__ __forceinline__ double sum_before(double v, double& total, Share<W>& s)
{
    const double mine = __ockl_wfscan_add_f64(v, true);
    if (lane() == 63)
        s.d[wave()] = mine;
    __syncthreads();
    double before = 0.0, t = 0.0;
    for (int w = 0; w < W; ++w) {
        if (w == wave())
            before = t;
        t += s.d[w];
    }
    __syncthreads();
    total = t;
    // (not mine - v, which rounds: what the lane before has)
    const double left = __shfl_up(mine, 1);
    return before + (lane() ? left : 0.0);
}
template <int W>
__device__ __forceinline__ unsigned long long sum_before(unsigned long long v, unsigned long long& total, Share<W>& s)
{
    const unsigned long long mine = __ockl_wfscan_add_u64(v, true);
    if (lane() == 63)
        s.u[wave()] = mine;
    __syncthreads();
    unsigned long long before = 0, t = 0;
    for (int w = 0; w < W; ++w) {
        if (w == wave())
            before = t;
        t += s.u[w];
    }
    __syncthreads();
    total = t;
    return before + mine - v;
}

} // namespace step
} // namespace mako
