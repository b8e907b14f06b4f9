// A workgroup on the CPU, for tests of device functions that talk across lanes: every thread of it is a context of its own, run in
// turn from one barrier or exchange to the next, in one thread of the process.  (Compiled by clang as C++, with this folder before
// the others that are searched for headers.)  What lanes exchange is there when all of a wave that have not ended have asked for
// it: code in which some lanes of a wave skip an exchange that others make is not for this.
#pragma once

#include <math.h>
#include <stddef.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <ucontext.h>

#include <type_traits>
#include <vector>

#define __host__
#define __device__
#define __global__
#define __forceinline__ inline
#define __launch_bounds__(...)
#define __shared__ thread_local // (static storage, which all lanes' contexts share)

struct dim3 {
    uint32_t x, y, z;
    dim3(uint32_t a = 1, uint32_t b = 1, uint32_t c = 1) : x(a), y(b), z(c) {}
};
typedef void* hipStream_t;
typedef int hipError_t;
constexpr int hipSuccess = 0, hipFuncAttributeMaxDynamicSharedMemorySize = 8;
inline hipError_t hipLaunchKernel(const void*, dim3, dim3, void**, size_t, hipStream_t)
{
    return 1; // (a test calls lanes::run() with a kernel's body)
}
inline hipError_t hipFuncSetAttribute(const void*, int, int)
{
    return 1;
}

inline dim3 threadIdx, blockIdx, blockDim, gridDim;

namespace lanes {

constexpr size_t kStack = 256 * 1024;

struct Gate { // of a wave, or of all
    uint32_t members = 0, arrived = 0, round = 0;
    uint64_t value[2][64], here[2] = {0, 0};
    void open()
    {
        arrived = 0;
        ++round;
        here[round & 1] = 0;
    }
    void left()
    {
        if (--members && arrived == members)
            open();
    }
};
struct Group {
    std::vector<ucontext_t> threads;
    std::vector<char> ended;
    std::vector<Gate> waves;
    Gate all;
    ucontext_t main;
    uint32_t running = 0;
    void (*body)(void*) = nullptr;
    void* arg = nullptr;
};
inline Group* group = nullptr;
inline std::vector<char> stacks; // (kept from one workgroup to the next)
inline bool backwards = false;   // the last thread first: what a barrier is missing for is seen by one of the orders

inline void yield()
{
    Group& g = *group;
    const uint32_t me = g.running;
    swapcontext(&g.threads[me], &g.main);
    g.running = me;
    threadIdx.x = me;
}
inline void wait(Gate& gate)
{
    const uint32_t round = gate.round;
    if (++gate.arrived == gate.members)
        gate.open();
    while (gate.round == round)
        yield();
}
inline void entry()
{
    Group& g = *group;
    g.body(g.arg);
    const uint32_t me = threadIdx.x;
    g.ended[me] = 1;
    g.waves[me / 64].left();
    g.all.left();
    swapcontext(&g.threads[me], &g.main);
}

// body() by every thread of a workgroup
template <class F>
void run(uint32_t threads, F body)
{
    Group g;
    group = &g;
    g.threads.resize(threads);
    if (stacks.size() < threads * kStack)
        stacks.resize(threads * kStack);
    g.ended.assign(threads, 0);
    g.waves.resize((threads + 63) / 64);
    g.all.members = threads;
    g.body = [](void* f) { (*static_cast<F*>(f))(); };
    g.arg = &body;
    blockDim.x = threads;
    for (uint32_t t = 0; t < threads; ++t) {
        ++g.waves[t / 64].members;
        getcontext(&g.threads[t]);
        g.threads[t].uc_stack.ss_sp = stacks.data() + t * kStack;
        g.threads[t].uc_stack.ss_size = kStack;
        g.threads[t].uc_link = nullptr;
        makecontext(&g.threads[t], entry, 0);
    }
    for (bool any = true; any;) {
        any = false;
        for (uint32_t i = 0; i < threads; ++i) {
            const uint32_t t = backwards ? threads - 1 - i : i;
            if (!g.ended[t]) {
                any = true;
                g.running = t;
                threadIdx.x = t;
                swapcontext(&g.main, &g.threads[t]);
            }
        }
    }
    group = nullptr;
}

// All lanes' values (and which lanes there are): they stay until the next exchange but one.
template <class T>
const uint64_t* exchange(T v, uint64_t* there = nullptr)
{
    static_assert(sizeof(T) <= 8, "a lane's value");
    Gate& w = group->waves[threadIdx.x / 64];
    const uint32_t at = w.round & 1, lane = threadIdx.x & 63;
    uint64_t bits = 0;
    __builtin_memcpy(&bits, &v, sizeof v);
    w.value[at][lane] = bits;
    w.here[at] |= 1ull << lane;
    wait(w);
    if (there)
        *there = w.here[at];
    return w.value[at];
}
template <class T>
T from(const uint64_t* values, uint32_t lane)
{
    T v;
    __builtin_memcpy(&v, values + lane, sizeof v);
    return v;
}
template <class T, class F>
T reduce(T v, F f)
{
    uint64_t there;
    const uint64_t* all = exchange(v, &there);
    bool first = true;
    for (uint32_t k = 0; k < 64; ++k)
        if (there >> k & 1) {
            v = first ? from<T>(all, k) : f(v, from<T>(all, k));
            first = false;
        }
    return v;
}
template <class T>
T scan(T v, bool inclusive)
{
    uint64_t there;
    const uint64_t* all = exchange(v, &there);
    const uint32_t lane = threadIdx.x & 63;
    T sum = 0;
    for (uint32_t k = 0; k < lane + (inclusive ? 1u : 0u); ++k)
        if (there >> k & 1)
            sum += from<T>(all, k);
    return sum;
}

} // namespace lanes

inline void __syncthreads()
{
    lanes::wait(lanes::group->all);
}
inline unsigned long long __ballot(int v)
{
    return lanes::reduce<unsigned long long>(v ? 1ull << (threadIdx.x & 63) : 0ull, [](unsigned long long a, unsigned long long b) { return a | b; });
}
template <class T>
T __shfl(T v, int lane)
{
    return lanes::from<T>(lanes::exchange(v), (uint32_t)lane & 63u);
}
template <class T>
T __shfl_up(T v, unsigned by)
{
    const uint32_t lane = threadIdx.x & 63;
    return lanes::from<T>(lanes::exchange(v), lane >= by ? lane - by : lane);
}
inline int lanes_first(int v)
{
    uint64_t there;
    const uint64_t* all = lanes::exchange(v, &there);
    return lanes::from<int>(all, (uint32_t)__builtin_ctzll(there));
}
inline uint32_t lanes_below(uint32_t mask, uint32_t lane)
{
    return (uint32_t)__builtin_popcount(lane >= 32 ? mask : mask & ((1u << lane) - 1u));
}
// (a wave's own number is the same in all its lanes, and is asked for where some skip it: no exchange)
#define __builtin_amdgcn_readfirstlane(v) (__builtin_strcmp(#v, "(int)(threadIdx.x >> 6)") == 0 ? (int)(threadIdx.x >> 6) : lanes_first((int)(v)))
#define __builtin_amdgcn_readlane(v, l) __shfl<int>(v, l)
#define __builtin_amdgcn_mbcnt_lo(mask, add) (lanes_below(mask, threadIdx.x & 63) + (add))
#define __builtin_amdgcn_mbcnt_hi(mask, add) ((threadIdx.x & 63) > 32 ? lanes_below(mask, (threadIdx.x & 63) - 32) + (add) : (add))
#define __builtin_amdgcn_logf(x) log2f(x)
#define __builtin_amdgcn_exp2f(x) exp2f(x)
#define __builtin_amdgcn_rcpf(x) (1.0f / (x))
#define __builtin_amdgcn_sqrtf(x) sqrtf(x)
#define __builtin_amdgcn_fence(...) ((void)lanes_first(0)) // (the lanes' writes before are there behind it)
#define __builtin_amdgcn_wave_barrier() ((void)lanes_first(0))
#define __builtin_amdgcn_sched_barrier(x) ((void)0)
inline int lanes_frexp_exp(double x)
{
    int e;
    (void)frexp(x, &e);
    return e;
}
#define __builtin_amdgcn_frexp_exp(x) lanes_frexp_exp(x)

extern "C" {
inline uint32_t __ockl_wfred_add_u32(uint32_t v) { return lanes::reduce(v, [](uint32_t a, uint32_t b) { return a + b; }); }
inline uint32_t __ockl_wfred_min_u32(uint32_t v) { return lanes::reduce(v, [](uint32_t a, uint32_t b) { return a < b ? a : b; }); }
inline uint32_t __ockl_wfred_max_u32(uint32_t v) { return lanes::reduce(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; }); }
inline float __ockl_wfred_max_f32(float v) { return lanes::reduce(v, [](float a, float b) { return fmaxf(a, b); }); }
inline double __ockl_wfred_add_f64(double v) { return lanes::reduce(v, [](double a, double b) { return a + b; }); }
inline uint32_t __ockl_wfscan_add_u32(uint32_t v, bool inclusive) { return lanes::scan(v, inclusive); }
inline double __ockl_wfscan_add_f64(double v, bool inclusive) { return lanes::scan(v, inclusive); }
inline uint64_t __ockl_wfscan_add_u64(uint64_t v, bool inclusive) { return lanes::scan(v, inclusive); }
}

inline int __popcll(unsigned long long v)
{
    return __builtin_popcountll(v);
}
inline float __uint_as_float(uint32_t u)
{
    return __builtin_bit_cast(float, u);
}
inline uint32_t __float_as_uint(float f)
{
    return __builtin_bit_cast(uint32_t, f);
}
template <class A, class B>
std::common_type_t<A, B> min(A a, B b)
{
    return (std::common_type_t<A, B>)b < (std::common_type_t<A, B>)a ? b : a;
}
template <class A, class B>
std::common_type_t<A, B> max(A a, B b)
{
    return (std::common_type_t<A, B>)a < (std::common_type_t<A, B>)b ? b : a;
}
template <class T, class V>
T atomicAdd(T* p, V v)
{
    const T was = *p;
    *p += (T)v;
    return was;
}
template <class T, class V>
T atomicMin(T* p, V v)
{
    const T was = *p;
    *p = was < (T)v ? was : (T)v;
    return was;
}
template <class T, class V>
T atomicMax(T* p, V v)
{
    const T was = *p;
    *p = was > (T)v ? was : (T)v;
    return was;
}
