// A workgroup on the host: enough of the HIP language for the kernels that the tests run without a GPU. Each thread of a
// workgroup is a context of its own; they take turns, and one runs until it waits for its wavefront (ballots, exchanges) or
// for the workgroup (__syncthreads). `first_wave` runs before the others wherever it can, so that what a barrier should
// order, and does not, comes out in the wrong order. One workgroup at a time; __shared__ is static.
#pragma once

#include <stdint.h>
#include <ucontext.h>

#include <algorithm>
#include <cmath>
#include <cstddef>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <vector>

#define __host__
#define __device__
#define __global__
#define __shared__ static
#define __forceinline__ inline
#define __noinline__ __attribute__((noinline))
#define __launch_bounds__(...)
#define __align__(n) __attribute__((aligned(n)))

struct dim3 {
    unsigned x, y, z;
    dim3(unsigned x_ = 1, unsigned y_ = 1, unsigned z_ = 1) : x(x_), y(y_), z(z_) {}
};
typedef int hipError_t;
typedef void *hipStream_t;
constexpr hipError_t hipSuccess = 0;
inline hipError_t hipGetLastError() { return hipSuccess; }

namespace host_gpu {

constexpr int WAVE = 64;

struct Thread {
    ucontext_t at;
    std::vector<char> stack;
    unsigned long waits_wave = 0, waits_all = 0;  // barriers that it has come to
    bool done = false;
};
struct Wave {
    uint64_t slots[WAVE];
    int arrived = 0;
    unsigned long passed = 0;
};
struct Workgroup {
    std::vector<Thread> threads;
    std::vector<Wave> waves;
    ucontext_t home;
    int now = 0, arrived = 0, finished = 0;
    unsigned long passed = 0;
    std::function<void()> body;
};
inline Workgroup *group = nullptr;
inline int first_wave = 0;
inline dim3 block_index, grid_size;

inline Thread &self() { return group->threads[group->now]; }
inline void yield() { swapcontext(&self().at, &group->home); }
inline void enter() {
    group->body();
    self().done = true;
    group->finished++;
    yield();
}
// Until all threads of the wavefront are here.
inline void meet_wave() {
    Wave &w = group->waves[group->now / WAVE];
    const unsigned long mine = ++self().waits_wave;
    if (++w.arrived == WAVE) {
        w.arrived = 0;
        w.passed++;
    }
    while (w.passed < mine) yield();
}
inline void meet_all() {
    Workgroup &g = *group;
    const unsigned long mine = ++self().waits_all;
    if (++g.arrived == (int)g.threads.size()) {
        g.arrived = 0;
        g.passed++;
    }
    while (g.passed < mine) yield();
}
// x of lane `from(lane)` of the wavefront, `other` where that is negative.
template <typename X, typename F>
X exchange(X x, X other, F from) {
    static_assert(sizeof(X) <= 8, "");
    const int lane = group->now % WAVE;
    Wave &w = group->waves[group->now / WAVE];
    memcpy(&w.slots[lane], &x, sizeof(X));
    meet_wave();
    const int at = from(lane);
    if (at >= 0) memcpy(&other, &w.slots[at], sizeof(X));
    meet_wave();
    return other;
}

// Runs the workgroup; false where threads wait for ones that are gone or wait elsewhere.
inline bool run(int threads, std::function<void()> body) {
    Workgroup g;
    g.threads.resize(threads);
    g.waves.resize(threads / WAVE);
    g.body = std::move(body);
    group = &g;
    for (Thread &t : g.threads) {
        t.stack.resize(1 << 16);
        getcontext(&t.at);
        t.at.uc_stack.ss_sp = t.stack.data();
        t.at.uc_stack.ss_size = t.stack.size();
        t.at.uc_link = &g.home;
        makecontext(&t.at, enter, 0);
    }
    const auto ready = [&](int i) {
        const Thread &t = g.threads[i];
        return !t.done && t.waits_all <= g.passed && t.waits_wave <= g.waves[i / WAVE].passed;
    };
    bool more = true;
    while (more) {
        more = false;
        for (size_t w = 0; w < g.waves.size() && !more; w++) {
            const int wave = ((int)w + first_wave) % (int)g.waves.size();
            for (int lane = 0; lane < WAVE; lane++) {
                if (!ready(wave * WAVE + lane)) continue;
                g.now = wave * WAVE + lane;
                swapcontext(&g.home, &g.threads[g.now].at);
                more = true;
            }
        }
    }
    group = nullptr;
    return g.finished == threads;
}

struct Index {
    struct X {
        operator unsigned() const { return group->now; }
    } x;
};
struct Block {
    struct X {
        operator unsigned() const { return block_index.x; }
    } x;
};
struct Grid {
    struct X {
        operator unsigned() const { return grid_size.x; }
    } x;
};
inline bool all_finished = true;

}  // namespace host_gpu

inline host_gpu::Index threadIdx;
inline host_gpu::Block blockIdx;
inline host_gpu::Grid gridDim;

#define hipLaunchKernelGGL(kernel, grid, block, lds, stream, ...)                                        \
    do {                                                                                                 \
        host_gpu::grid_size = grid;                                                                      \
        for (unsigned b_ = 0; b_ < host_gpu::grid_size.x; b_++) {                                        \
            host_gpu::block_index = dim3(b_);                                                            \
            if (!host_gpu::run((int)(block).x, [&] { kernel(__VA_ARGS__); })) host_gpu::all_finished = false; \
        }                                                                                                \
    } while (0)

inline void __syncthreads() { host_gpu::meet_all(); }
inline unsigned long long __ballot(int x) {
    unsigned long long r = 0;
    const int lane = host_gpu::group->now % host_gpu::WAVE;
    host_gpu::Wave &w = host_gpu::group->waves[host_gpu::group->now / host_gpu::WAVE];
    w.slots[lane] = x != 0;
    host_gpu::meet_wave();
    for (int i = 0; i < host_gpu::WAVE; i++) r |= (unsigned long long)w.slots[i] << i;
    host_gpu::meet_wave();
    return r;
}
template <typename X>
X __shfl_xor(X x, int by) {
    return host_gpu::exchange(x, x, [&](int lane) { return lane ^ by; });
}
// The controls that shift within rows of 16 (0x111 on) or the wavefront (0x138) or hand on a row's or half's last lane.
inline int __builtin_amdgcn_update_dpp(int other, int x, int control, int rows, int, bool) {
    return host_gpu::exchange(x, other, [&](int lane) {
        const int row = lane / 16;
        if (!(rows >> row & 1)) return -1;
        if (control > 0x110 && control < 0x120) return lane % 16 >= control - 0x110 ? lane - (control - 0x110) : -1;
        if (control == 0x138) return lane - 1;
        if (control == 0x142) return row * 16 - 1;
        if (control == 0x143) return row >= 2 ? 31 : -1;
        abort();
    });
}
inline int __builtin_amdgcn_readlane(int x, int from) {
    return host_gpu::exchange(x, x, [&](int) { return from; });
}
inline double __builtin_amdgcn_fract(double x) { return x - std::floor(x); }
inline int __builtin_amdgcn_frexp_exp(double x) {
    int e = 0;
    if (std::isfinite(x)) std::frexp(x, &e);
    return e;
}
inline uint32_t __builtin_amdgcn_perm(uint32_t, uint32_t, uint32_t) { abort(); }

template <typename X>
X atomicAdd(X *at, X by) {
    const X old = *at;
    *at += by;
    return old;
}
inline int atomicMin(int *at, int x) {
    const int old = *at;
    *at = std::min(old, x);
    return old;
}
inline uint32_t __float_as_uint(float x) { return __builtin_bit_cast(uint32_t, x); }
inline float __uint_as_float(uint32_t x) { return __builtin_bit_cast(float, x); }
inline float __log2f(float x) { return std::log2(x); }
inline float __builtin_amdgcn_exp2f(float x) { return std::exp2(x); }
template <typename X, typename Y>
auto min(X x, Y y) {
    return y < x ? y : x;
}
template <typename X, typename Y>
auto max(X x, Y y) {
    return x < y ? y : x;
}
