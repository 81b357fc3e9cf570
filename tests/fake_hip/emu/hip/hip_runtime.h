// A stand-in for <hip/hip_runtime.h> under which kernels run on the CPU, one workgroup at a time, a thread of the workgroup being a fiber:
// barriers and lane exchanges hand over to the next fiber until all that take part have arrived.  For checks of what a kernel reads and writes
// (tests/test_kernel_bounds_cpu.py): TEST INFRASTRUCTURE ONLY.  Not for timing, and not a model of the memory system -- a missing wait is not
// seen here, a missing barrier mostly is.
#pragma once
#include "../../hip/hip_runtime.h"

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <memory>
#include <tuple>
#include <vector>

#define __global__
#define __device__
#define __host__
#define __shared__ static
#define __forceinline__ inline
#define __launch_bounds__(...)

struct dim3 {
    uint32_t x, y, z;
    dim3(uint32_t x_ = 1, uint32_t y_ = 1, uint32_t z_ = 1) : x(x_), y(y_), z(z_) {}
};

namespace emu {

struct group {                      // threads that meet: `size` of them while none has ended
    int size = 0, arrived = 0;
    uint64_t generation = 0;
    void look() { if (size && arrived == size) { arrived = 0; ++generation; } }
};
struct fiber {
    void *sp = nullptr;
    uint32_t id = 0;
    bool done = false;
};
// saves the callee's registers and the stack pointer, goes on where `to` was saved (x86-64; without the system calls of swapcontext)
extern "C" void emu_switch(void **from, void *to);
asm(R"(
.weak emu_switch
.type emu_switch,@function
emu_switch:
    pushq %rbp
    pushq %rbx
    pushq %r12
    pushq %r13
    pushq %r14
    pushq %r15
    movq %rsp, (%rdi)
    movq %rsi, %rsp
    popq %r15
    popq %r14
    popq %r13
    popq %r12
    popq %rbx
    popq %rbp
    ret
)");
inline dim3 block_idx, grid_dim;
inline const void *kernarg = nullptr;          // the kernel's first argument
inline void *scheduler = nullptr;
inline fiber *current = nullptr;
inline const std::function<void()> *body = nullptr;
inline group whole;
inline std::vector<group> waves, rows, quads;  // 64, 16 and 4 lanes
inline std::vector<uint64_t> lanes;            // what a thread shows the others
inline std::vector<fiber> fibers;
inline std::vector<char> stacks;
constexpr size_t STACK = 256 << 10;

inline void yield() { emu_switch(&current->sp, scheduler); }
inline void meet(group &g)
{
    const uint64_t seen = g.generation;
    ++g.arrived;
    g.look();
    while (g.generation == seen) yield();
}
inline group &group_of(int width)
{
    const uint32_t t = current->id;
    return width == 64 ? waves[t / 64] : width == 16 ? rows[t / 16] : quads[t / 4];
}
template <class T>
T exchange(T v, uint32_t from_lane, int width)          // the value of that lane of this wave; `width` lanes take part
{
    static_assert(sizeof(T) <= 8);
    uint64_t bits = 0;
    memcpy(&bits, &v, sizeof v);
    lanes[current->id] = bits;
    meet(group_of(width));
    bits = lanes[current->id / 64 * 64 + from_lane];
    meet(group_of(width));
    memcpy(&v, &bits, sizeof v);
    return v;
}
inline void entry()
{
    (*body)();
    fiber &f = *current;
    f.done = true;
    for (group *g : {&whole, &waves[f.id / 64], &rows[f.id / 16], &quads[f.id / 4]}) { --g->size; g->look(); }
    yield();
    abort();
}
inline void run_workgroup(uint32_t threads)
{
    if (fibers.size() < threads) { fibers.resize(threads); stacks.resize(threads * STACK); }
    whole = group{(int)threads};
    waves.assign((threads + 63) / 64, {}), rows.assign((threads + 15) / 16, {}), quads.assign((threads + 3) / 4, {});
    lanes.assign((threads + 63) / 64 * 64, 0);
    for (uint32_t t = 0; t < threads; ++t) {
        ++waves[t / 64].size, ++rows[t / 16].size, ++quads[t / 4].size;
        fiber &f = fibers[t];
        f.id = t, f.done = false;
        // an empty frame under entry(): six registers, its address, and a return address that is never used (the stack is 16-byte aligned at a call)
        void **top = reinterpret_cast<void **>((reinterpret_cast<uintptr_t>(stacks.data()) + (t + 1) * STACK) & ~uintptr_t(63));
        top -= 8;
        memset(top, 0, 8 * sizeof(void *));
        top[6] = reinterpret_cast<void *>(entry);
        f.sp = top;
    }
    for (bool more = true; more;) {
        more = false;
        for (uint32_t t = 0; t < threads; ++t) {
            if (fibers[t].done) continue;
            more = true;
            current = &fibers[t];
            emu_switch(&scheduler, current->sp);
        }
    }
}
template <class... P, class... A>
void launch(void (*kernel)(P...), dim3 grid, dim3 block, A... args)
{
    if ((uint64_t)grid.x * grid.y * grid.z * block.x >= 1ull << 32 || grid.y > 65535 || grid.z > 65535 || block.x > 1024) { printf("launch limits\n"); abort(); }
    std::tuple<std::decay_t<P>...> kept(args...);
    kernarg = &std::get<0>(kept);
    const std::function<void()> f = [&] { std::apply(kernel, kept); };
    body = &f;
    grid_dim = grid;
    for (uint32_t z = 0; z < grid.z; ++z)
        for (uint32_t y = 0; y < grid.y; ++y)
            for (uint32_t x = 0; x < grid.x; ++x) {
                block_idx = dim3(x, y, z);
                run_workgroup(block.x);
            }
}

// D = A B + C over a wave, K values of k a lane pair: A[i = lane % 32][k], B[k][j = lane % 32], k = KL (lane / 32) + e; register r of lane l is
// D[8 (r / 4) + 4 (l / 32) + r % 4][l % 32]
template <int KL, class V, class C>
C mfma_32x32(const V &a, const V &b, C c)
{
    static std::vector<float> all;
    const uint32_t t = current->id, wave = t / 64, lane = t % 64;
    if (all.size() < waves.size() * 64 * 16) all.resize(waves.size() * 64 * 16);
    float *mine = all.data() + (wave * 64 + lane) * 16;
    for (int e = 0; e < KL; ++e) mine[e] = a[e], mine[8 + e] = b[e];
    meet(waves[wave]);
    for (int r = 0; r < 16; ++r) {
        const int i = 8 * (r / 4) + 4 * (lane / 32) + r % 4, j = lane % 32;
        float s = c[r];
        for (int h = 0; h < 2; ++h)
            for (int e = 0; e < KL; ++e) s += all[(wave * 64 + h * 32 + i) * 16 + e] * all[(wave * 64 + h * 32 + j) * 16 + 8 + e];
        c[r] = s;
    }
    meet(waves[wave]);
    return c;
}

}  // namespace emu

struct emu_thread_idx {
    struct { operator uint32_t() const { return emu::current->id; } } x;
};
inline emu_thread_idx threadIdx;
#define blockIdx emu::block_idx
#define gridDim emu::grid_dim
#define hipLaunchKernelGGL(kernel, grid, block, lds, stream, ...) emu::launch(kernel, grid, block, __VA_ARGS__)

inline void __syncthreads() { emu::meet(emu::whole); }
inline void emu_wave_sync() { emu::meet(emu::waves[emu::current->id / 64]); }
inline bool __all(int p)
{
    emu::lanes[emu::current->id] = p;
    emu_wave_sync();
    bool all = true;
    for (int i = 0; i < 64; ++i) all = all && emu::lanes[emu::current->id / 64 * 64 + i];
    emu_wave_sync();
    return all;
}
template <class T> T __shfl_xor(T v, int mask, int) { return emu::exchange(v, (emu::current->id & 63) ^ mask, 64); }
inline int __builtin_amdgcn_update_dpp_(int, int v, int ctrl, int, int, bool)
{
    const uint32_t l = emu::current->id & 63;
    if (ctrl == 0xB1) return emu::exchange(v, l ^ 1, 4);
    if (ctrl == 0x4E) return emu::exchange(v, l ^ 2, 4);
    if (ctrl == 0x141) return emu::exchange(v, l ^ 7, 16);
    if (ctrl == 0x140) return emu::exchange(v, l ^ 15, 16);
    abort();
}
#define __builtin_amdgcn_update_dpp __builtin_amdgcn_update_dpp_
#define __builtin_amdgcn_exp2f(x) exp2f(x)
#define __builtin_amdgcn_rcpf(x) (1.0f / (x))
#define __builtin_amdgcn_sched_barrier(x) ((void)0)
#define __builtin_amdgcn_readfirstlane(x) (x)
#define __builtin_amdgcn_kernarg_segment_ptr() emu::kernarg
#define __builtin_amdgcn_cvt_pk_fp8_f32(a, b, old, hi) ((hi) ? (int)(((uint32_t)(old) & 0xFFFFu) | 0x38380000u) : (int)(((uint32_t)(old) & 0xFFFF0000u) | 0x3838u))
#define __builtin_amdgcn_cvt_pk_bf8_f32 __builtin_amdgcn_cvt_pk_fp8_f32
#define __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, ...) emu::mfma_32x32<8>(a, b, c)
#define __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, ...) emu::mfma_32x32<8>(a, b, c)
#define __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, ...) emu::mfma_32x32<1>(&(const float &)(a), &(const float &)(b), c)
inline float __uint_as_float(uint32_t u) { float f; memcpy(&f, &u, 4); return f; }
inline uint32_t __float_as_uint(float f) { uint32_t u; memcpy(&u, &f, 4); return u; }
inline float rsqrtf(float x) { return 1.0f / sqrtf(x); }
template <class T> T min(T a, T b) { return b < a ? b : a; }
template <class T> T max(T a, T b) { return a < b ? b : a; }
