// A workgroup on the CPU, for tests of a kernel's own control flow: every lane is a
// fiber of one thread, barriers and cross-lane operations are where fibers take turns,
// shared memory is static.  Found by a host compile of a kernel's source in the place of
// the HIP header; has what the sampler's kernels use.  A workgroup that passes more
// barriers than it is allowed, or whose lanes wait for each other, is given up.
#pragma once
#include <math.h>
#include <stdint.h>
#include <string.h>
#include <ucontext.h>

#include <functional>
#include <vector>

namespace host_gpu {

struct Index {
    uint32_t x, y, z;
};

struct Fiber {
    ucontext_t at;
    std::vector<char> stack;
    bool done = false;
    uint64_t passed[2] = {0, 0};  // barriers of the wave and of the workgroup
};

enum End { kEnded, kTooLong, kStuck };

struct Group {
    std::vector<Fiber> lanes;
    ucontext_t scheduler;
    uint32_t now = 0;
    Index block;
    std::vector<uint64_t> cell;  // a value a lane, for the cross-lane operations
    std::function<void()> body;
};
inline Group* group = nullptr;

__attribute__((noinline)) inline Index thread_index() { return {group->now, 0, 0}; }
__attribute__((noinline)) inline Index block_index() { return group->block; }

__attribute__((noinline)) inline void turn() { swapcontext(&group->lanes[group->now].at, &group->scheduler); }

// Waits for the lanes of the wave (64) or of the whole workgroup.
inline void barrier(int whole) {
    Group& g = *group;
    const uint32_t n = static_cast<uint32_t>(g.lanes.size()), from = whole ? 0 : g.now / 64 * 64, to = whole ? n : from + 64;
    const uint64_t mine = ++g.lanes[g.now].passed[whole];
    for (;;) {
        bool all = true;
        for (uint32_t i = from; i < to && all; i++) all = g.lanes[i].done || g.lanes[i].passed[whole] >= mine;
        if (all) return;
        turn();
    }
}

template <class F>
uint64_t exchange(uint64_t v, const F& read) {
    Group& g = *group;
    const uint32_t lane = g.now;
    g.cell[lane] = v;
    barrier(0);
    const uint64_t r = read(&g.cell[lane / 64 * 64], lane % 64);
    barrier(0);
    return r;
}

inline void enter() {
    Group& g = *group;
    g.body();
    g.lanes[g.now].done = true;
    turn();
}

// Runs a workgroup; `most` barriers of the workgroup and of each wave at most.
inline End run(uint32_t threads, Index block, uint64_t most, std::function<void()> body) {
    Group g;
    g.lanes.resize(threads);
    g.cell.resize(threads);
    g.block = block;
    g.body = std::move(body);
    group = &g;
    for (Fiber& f : g.lanes) {
        f.stack.resize(64 << 10);
        getcontext(&f.at);
        f.at.uc_stack.ss_sp = f.stack.data();
        f.at.uc_stack.ss_size = f.stack.size();
        f.at.uc_link = nullptr;
        makecontext(&f.at, enter, 0);
    }
    for (;;) {
        bool live = false;
        uint64_t before = 0, after = 0, longest = 0;
        for (uint32_t i = 0; i < threads; i++) {
            Fiber& f = g.lanes[i];
            before += f.passed[0] + f.passed[1];
            if (!f.done) {
                g.now = i;
                swapcontext(&g.scheduler, &f.at);
            }
            live = live || !f.done;
            after += f.passed[0] + f.passed[1] + f.done;
            longest = f.passed[0] > longest ? f.passed[0] : longest;
            longest = f.passed[1] > longest ? f.passed[1] : longest;
        }
        if (!live) return kEnded;
        if (longest > most) return kTooLong;
        if (after == before) return kStuck;
    }
}

inline uint32_t dpp(uint32_t old, uint32_t v, int ctrl, int rows) {
    return static_cast<uint32_t>(exchange(v, [&](const uint64_t* c, uint32_t lane) -> uint64_t {
        if (!(rows >> (lane / 16) & 1)) return old;
        if (ctrl > 0x110 && ctrl < 0x120) {  // shifted within the row
            const uint32_t n = ctrl & 15;
            return lane % 16 >= n ? c[lane - n] : old;
        }
        if (ctrl == 0x142) return lane >= 16 ? c[lane / 16 * 16 - 1] : old;  // the row before's last
        if (ctrl == 0x143) return lane >= 32 ? c[31] : old;                  // the lower half's last
        __builtin_trap();
    }));
}

template <class T>
T add(T* p, T v) {
    const T was = *p;
    *p = was + v;
    return was;
}

}  // namespace host_gpu

#define __global__
#define __device__
#define __forceinline__ inline
#define __launch_bounds__(...)
#define __shared__ static
#define threadIdx (host_gpu::thread_index())
#define blockIdx (host_gpu::block_index())
#define asm(...)

struct ulonglong2 {
    unsigned long long x, y;
};

inline void __syncthreads() { host_gpu::barrier(1); }
inline uint64_t __ballot(bool v) {
    return host_gpu::exchange(v, [](const uint64_t* c, uint32_t) {
        uint64_t m = 0;
        for (int i = 0; i < 64; i++) m |= c[i] << i;
        return m;
    });
}
inline uint32_t __shfl_xor(uint32_t v, int o) {
    return static_cast<uint32_t>(host_gpu::exchange(v, [&](const uint64_t* c, uint32_t lane) { return c[lane ^ o]; }));
}
inline int host_readlane(int v, uint32_t from) {
    return static_cast<int>(host_gpu::exchange(static_cast<uint32_t>(v), [&](const uint64_t* c, uint32_t) { return c[from & 63]; }));
}
#define __builtin_amdgcn_readlane(v, from) host_readlane(v, from)
#define __builtin_amdgcn_update_dpp(old, v, ctrl, rows, banks, bound) \
    static_cast<int>(host_gpu::dpp(static_cast<uint32_t>(old), static_cast<uint32_t>(v), ctrl, rows))

inline uint32_t atomicAdd(uint32_t* p, uint32_t v) { return host_gpu::add(p, v); }
inline unsigned long long atomicAdd(unsigned long long* p, unsigned long long v) { return host_gpu::add(p, v); }
inline uint32_t atomicOr(uint32_t* p, uint32_t v) {
    const uint32_t was = *p;
    *p = was | v;
    return was;
}

template <class T>
T min(T a, T b) { return b < a ? b : a; }
template <class T>
T max(T a, T b) { return a < b ? b : a; }
