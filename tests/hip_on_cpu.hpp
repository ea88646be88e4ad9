// Kernels on the CPU: stands in for paged.hpp where a test compiles a kernel's source
// with a host compiler, to follow its reads and writes before a GPU runs it.  Threads
// are fibers of one process that change places at barriers; a wave's 64 trade values
// at a barrier of their own.  Blocks run one after another, so that __shared__ is static.
// What ends with every thread waiting says so and aborts.
#pragma once

#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <ucontext.h>

#include <functional>
#include <vector>

#include "lmx/paged.h"
#include "paged_index.hpp"

#define __global__
#define __device__
#define __forceinline__ inline
#define __shared__ static
#define __launch_bounds__(...)

struct dim3 {
    unsigned x, y, z;
    dim3(unsigned x = 1, unsigned y = 1, unsigned z = 1) : x(x), y(y), z(z) {}
};
typedef void* hipStream_t;
inline int hipGetLastError() { return 0; }
#define LMX_CHECK_LAUNCH() (void)0

namespace on_cpu {

struct Barrier {
    int here = 0, of = 0;
    long gen = 0;
};
struct Fiber {
    ucontext_t at;
    dim3 thread;
    bool done = false;
    int wave = 0, lane = 0;
    std::vector<char> stack;
};
struct Block {
    std::vector<Fiber> fibers;
    std::vector<Barrier> waves;
    std::vector<std::vector<int64_t>> lanes;  // what a wave's lanes show each other
    Barrier all;
    ucontext_t main;
    Fiber* now = nullptr;
    dim3 block;
    long steps = 0;  // barriers passed and threads ended
};
inline Block* cur = nullptr;

inline void pass_if_full(Barrier& b) {
    if (b.of && b.here == b.of) {
        b.here = 0;
        ++b.gen;
        ++cur->steps;
    }
}
inline void wait(Barrier& b) {
    const long gen = b.gen;
    ++b.here;
    pass_if_full(b);
    while (b.gen == gen) swapcontext(&cur->now->at, &cur->main);
}

inline const std::function<void()>* body = nullptr;
inline void start() {
    (*body)();
    Fiber* f = cur->now;
    f->done = true;
    ++cur->steps;
    for (Barrier* b : {&cur->all, &cur->waves[f->wave]}) {  // the others wait for it no more
        --b->of;
        pass_if_full(*b);
    }
    swapcontext(&f->at, &cur->main);
}

inline void launch(dim3 grid, dim3 block, const std::function<void()>& kernel) {
    body = &kernel;
    const int n = (int)(block.x * block.y * block.z);
    for (unsigned z = 0; z < grid.z; ++z)
        for (unsigned y = 0; y < grid.y; ++y)
            for (unsigned x = 0; x < grid.x; ++x) {
                Block b;
                cur = &b;
                b.block = dim3(x, y, z);
                b.fibers.resize(n);
                b.waves.resize((n + 63) / 64);
                b.lanes.assign((n + 63) / 64, std::vector<int64_t>(64));
                b.all.of = n;
                for (int i = 0; i < n; ++i) {
                    Fiber& f = b.fibers[i];
                    f.thread = dim3(i % block.x, i / block.x % block.y, i / block.x / block.y);
                    f.wave = i / 64;
                    f.lane = i % 64;
                    ++b.waves[f.wave].of;
                    f.stack.resize(1 << 15);
                    getcontext(&f.at);
                    f.at.uc_stack.ss_sp = f.stack.data();
                    f.at.uc_stack.ss_size = f.stack.size();
                    f.at.uc_link = nullptr;
                    makecontext(&f.at, start, 0);
                }
                for (bool more = true; more;) {
                    more = false;
                    const long before = b.steps;
                    for (Fiber& f : b.fibers)
                        if (!f.done) {
                            more = true;
                            b.now = &f;
                            swapcontext(&b.main, &f.at);
                        }
                    if (more && b.steps == before) {
                        printf("every thread waits\n");
                        abort();
                    }
                }
            }
    cur = nullptr;
}

// The value of lane `from` of the caller's wave, of which all lanes take part.
template <typename T>
T of_lane(T x, int from) {
    Fiber* f = cur->now;
    auto& v = cur->lanes[f->wave];
    v[f->lane] = 0;
    memcpy(&v[f->lane], &x, sizeof x);
    wait(cur->waves[f->wave]);
    T y;
    memcpy(&y, &v[from], sizeof y);
    wait(cur->waves[f->wave]);
    return y;
}

}  // namespace on_cpu

#define threadIdx (on_cpu::cur->now->thread)
#define blockIdx (on_cpu::cur->block)
#define hipLaunchKernelGGL(kernel, grid, block, lds, stream, ...) on_cpu::launch(grid, block, [&] { kernel(__VA_ARGS__); })
inline void __syncthreads() { on_cpu::wait(on_cpu::cur->all); }
template <typename T>
T __shfl_up(T x, int d, int) {
    const int lane = on_cpu::cur->now->lane;
    return on_cpu::of_lane(x, lane >= d ? lane - d : lane);
}
