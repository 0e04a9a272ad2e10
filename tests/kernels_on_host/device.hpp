// device.hpp - gfx950 kernel sources compiled for the host and run there: what
// the paged kernels and the log probabilities use of a device, so that their own
// index arithmetic runs under AddressSanitizer.
//
// A block's threads are fibers of one host thread.  A lane operation (a read of
// another lane, a ballot, a matrix product) waits until every lane of the wave
// that has not ended waits in one, which has to be the same: lanes that part are
// an error here.  Blocks run one after the other, a block's waves each as far as it
// comes without a barrier; or, backwards, the last wave first and all of them in turn
// by one lane operation, so that what a missing barrier leaves to chance comes out in
// two ways.  Static LDS arrays are static arrays, dynamic LDS is an allocation of the
// launch's size.
#pragma once

#include <math.h>
#include <stddef.h>
#include <stdint.h>

#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <utility>

#define __device__
#define __host__
#define __global__
#define __forceinline__ inline
#define __launch_bounds__(...)
#define __shared__ static

using std::max;
using std::min;

struct alignas(8) float2 {
    float x, y;
};
struct alignas(16) float4 {
    float x, y, z, w;
};
struct alignas(16) int4 {
    int x, y, z, w;
};
struct alignas(16) uint4 {
    uint32_t x, y, z, w;
};
inline float2 make_float2(float x, float y) { return {x, y}; }
inline float4 make_float4(float x, float y, float z, float w) { return {x, y, z, w}; }
inline int4 make_int4(int x, int y, int z, int w) { return {x, y, z, w}; }
inline uint4 make_uint4(uint32_t x, uint32_t y, uint32_t z, uint32_t w) { return {x, y, z, w}; }

struct dim3 {
    unsigned x, y, z;
    dim3(unsigned x_ = 1, unsigned y_ = 1, unsigned z_ = 1) : x(x_), y(y_), z(z_) {}
};
typedef int hipError_t;
typedef void* hipStream_t;
constexpr hipError_t hipSuccess = 0, hipErrorInvalidConfiguration = 9;
constexpr int hipFuncAttributeMaxDynamicSharedMemorySize = 8;
inline const char* hipGetErrorString(hipError_t) { return "host"; }
inline hipError_t hipGetLastError() { return hipSuccess; }
inline hipError_t hipPeekAtLastError() { return hipSuccess; }
inline hipError_t hipFuncSetAttribute(const void*, int, int) { return hipSuccess; }

namespace host {

constexpr int kLanes = 64;
constexpr size_t kStack = 256 * 1024;
typedef void (*LaneOp)(void** lanes);  // the lanes' operands, null where a lane has ended

enum State { kReady, kLaneOp, kBarrier, kEnded };
struct Thread {
    void* sp;
    char* stack;
    State state;
    LaneOp op;
    void* operand;
};

inline Thread* threads;  // of the block
inline Thread* now;      // that runs
inline void* scheduler;  // its stack pointer
inline dim3 thread_idx, block_idx, grid_dim, block_dim;
inline char* dynamic_lds;
inline size_t dynamic_bytes;
inline std::function<void()>* body;
inline int order = 1;  // of blocks and waves: 1, or -1

extern "C" void host_switch(void** save, void* to);
asm(R"(
.text
.weak host_switch
.type host_switch, @function
host_switch:
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

[[noreturn]] inline void fail(const char* what) {
    std::fprintf(stderr, "kernels on the host: %s (block %u %u %u, thread %u)\n", what, block_idx.x, block_idx.y, block_idx.z, thread_idx.x);
    std::abort();
}

inline void wait_as(State s) {
    now->state = s;
    host_switch(&now->sp, scheduler);
}
inline void entry() {
    (*body)();
    wait_as(kEnded);
    fail("a thread went on after its end");
}

// The block's threads until all have ended.
inline void run_block(int n) {
    for (int i = 0; i < n; ++i) {
        Thread& t = threads[i];
        t.state = kReady;
        void** top = reinterpret_cast<void**>(t.stack + kStack - 64);
        *--top = nullptr;  // (a call's return address: the stack is 16-byte aligned before it)
        *--top = reinterpret_cast<void*>(&entry);
        for (int r = 0; r < 6; ++r) *--top = nullptr;
        t.sp = top;
    }
    for (;;) {
        int ended = 0, at_barrier = 0;
        const int waves = (n + kLanes - 1) / kLanes;
        for (int wave = 0; wave < waves; ++wave) {
            const int w = (order > 0 ? wave : waves - 1 - wave) * kLanes, lanes = std::min(kLanes, n - w);
            for (bool again = true; again;) {
                again = order > 0;
                for (int i = w; i < w + lanes; ++i)
                    if (threads[i].state == kReady) {
                        now = &threads[i];
                        thread_idx = dim3(i, 0, 0);
                        host_switch(&scheduler, now->sp);
                    }
                void* operands[kLanes] = {};
                const Thread* first = nullptr;
                bool parted = false;
                for (int i = 0; i < lanes; ++i) {
                    Thread& t = threads[w + i];
                    if (t.state != kLaneOp) continue;
                    if (!first) first = &t;
                    parted |= t.op != first->op;
                    operands[i] = t.operand;
                }
                if (!first) break;
                for (int i = 0; i < lanes; ++i) parted |= threads[w + i].state == kBarrier;
                if (parted) fail("lanes of a wave in different operations");
                first->op(operands);
                for (int i = 0; i < lanes; ++i)
                    if (threads[w + i].state == kLaneOp) threads[w + i].state = kReady;
            }
            for (int i = 0; i < lanes; ++i) {
                ended += threads[w + i].state == kEnded;
                at_barrier += threads[w + i].state == kBarrier;
            }
        }
        if (ended == n) return;
        if (ended + at_barrier == n)
            for (int i = 0; i < n; ++i)
                if (threads[i].state == kBarrier) threads[i].state = kReady;
    }
}

constexpr int kMostThreads = 1024;
template <typename Kernel, typename... Args>
void launch(Kernel kernel, dim3 grid, dim3 block, size_t lds, hipStream_t, const Args&... args) {
    static Thread all[kMostThreads];
    const int n = static_cast<int>(block.x);
    if (n > kMostThreads || block.y != 1 || block.z != 1) fail("block size");
    for (int i = 0; i < n; ++i)
        if (!all[i].stack) all[i].stack = static_cast<char*>(std::aligned_alloc(64, kStack));
    threads = all;
    grid_dim = grid;
    block_dim = block;
    std::function<void()> run = [&] { kernel(args...); };
    body = &run;
    const int64_t blocks = static_cast<int64_t>(grid.x) * grid.y * grid.z;
    for (int64_t i = 0; i < blocks; ++i) {
        const int64_t b = order > 0 ? i : blocks - 1 - i;
        block_idx = dim3(static_cast<unsigned>(b % grid.x), static_cast<unsigned>(b / grid.x % grid.y), static_cast<unsigned>(b / grid.x / grid.y));
        dynamic_bytes = lds;
        dynamic_lds = lds ? static_cast<char*>(std::aligned_alloc(64, (lds + 63) / 64 * 64)) : nullptr;
        if (lds) std::memset(dynamic_lds, 0xA5, lds);
        run_block(n);
        std::free(dynamic_lds);
    }
}

// `op` over the lanes' operands T, in each lane
template <typename T>
inline void together(LaneOp op, T& operand) {
    now->op = op;
    now->operand = &operand;
    wait_as(kLaneOp);
}

struct FromLane {
    uint64_t in, out;
    int lane;  // read from
};
inline uint64_t from_lane(uint64_t v, int lane) {
    FromLane f{v, 0, lane};
    together(
        [](void** lanes) {
            for (int i = 0; i < kLanes; ++i) {
                FromLane* f = static_cast<FromLane*>(lanes[i]);
                if (!f) continue;
                const FromLane* g = static_cast<FromLane*>(lanes[f->lane & (kLanes - 1)]);
                f->out = g ? g->in : 0;
            }
        },
        f);
    return f.out;
}
inline int lane_id() { return static_cast<int>(thread_idx.x % kLanes); }

struct Ballot {
    bool in;
    uint64_t out;
};
inline uint64_t ballot(bool v) {
    Ballot b{v, 0};
    together(
        [](void** lanes) {
            uint64_t all = 0;
            for (int i = 0; i < kLanes; ++i)
                if (lanes[i] && static_cast<Ballot*>(lanes[i])->in) all |= uint64_t(1) << i;
            for (int i = 0; i < kLanes; ++i)
                if (lanes[i]) static_cast<Ballot*>(lanes[i])->out = all;
        },
        b);
    return b.out;
}
struct First {
    int in, out;
};
inline int readfirstlane(int v) {
    First f{v, 0};
    together(
        [](void** lanes) {
            int i = 0;
            while (!lanes[i]) ++i;
            const int v = static_cast<First*>(lanes[i])->in;
            for (; i < kLanes; ++i)
                if (lanes[i]) static_cast<First*>(lanes[i])->out = v;
        },
        f);
    return f.out;
}
// data parallel primitives: within rows of 16 lanes
inline int update_dpp(int old, int v, int ctrl, int, int, bool bound) {
    const int lane = lane_id(), row = lane & ~15, i = lane & 15;
    int from = -1;
    if (ctrl < 0x100)
        from = (lane & ~3) | (ctrl >> 2 * (lane & 3) & 3);
    else if (ctrl > 0x110 && ctrl < 0x120)
        from = i >= ctrl - 0x110 ? lane - (ctrl - 0x110) : -1;
    else if (ctrl > 0x120 && ctrl < 0x130)
        from = row | ((i - (ctrl - 0x120)) & 15);
    else if (ctrl == 0x140)
        from = row | (15 - i);
    else if (ctrl == 0x141)
        from = (lane & ~7) | (7 - (lane & 7));
    else
        fail("lane move");
    const int got = static_cast<int>(from_lane(static_cast<uint32_t>(v), from < 0 ? lane : from));
    return from < 0 ? (bound ? 0 : old) : got;
}
struct Pair {
    uint32_t v[2];
    uint32_t operator[](int i) const { return v[i]; }
};
// odd blocks of N lanes of a and even ones of b change places
template <int N>
inline Pair swap_rows(uint32_t a, uint32_t b) {
    const int lane = lane_id();
    const bool odd = lane / N & 1;
    const uint64_t other = from_lane(static_cast<uint64_t>(b) << 32 | a, lane ^ N);
    return odd ? Pair{{static_cast<uint32_t>(other >> 32), b}} : Pair{{a, static_cast<uint32_t>(other)}};
}

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef float float16_t __attribute__((ext_vector_type(16)));
template <int N, typename C>
struct Product {
    half8_t a, b;
    C c;
};
// D = A B + C: lane l has A's row l % N and B's column l % N, eight of the depth from 8 (l / N) on; of C and D column l % N,
// four rows in a row at a time
template <int N, typename C, int ELEMENTS>
inline C product(half8_t a, half8_t b, C c) {
    Product<N, C> p{a, b, c};
    together(
        [](void** lanes) {
            constexpr int kDepth = 8 * (kLanes / N);
            static float A[N][kDepth], B[N][kDepth];
            for (int l = 0; l < kLanes; ++l) {
                if (!lanes[l]) fail("a matrix product without all lanes");
                const auto* p = static_cast<Product<N, C>*>(lanes[l]);
                for (int e = 0; e < 8; ++e) {
                    A[l % N][8 * (l / N) + e] = static_cast<float>(p->a[e]);
                    B[l % N][8 * (l / N) + e] = static_cast<float>(p->b[e]);
                }
            }
            for (int l = 0; l < kLanes; ++l) {
                auto* p = static_cast<Product<N, C>*>(lanes[l]);
                for (int v = 0; v < ELEMENTS; ++v) {
                    const int row = v / 4 * (4 * (kLanes / N)) + 4 * (l / N) + v % 4;
                    float s = p->c[v];
                    for (int k = 0; k < kDepth; ++k) s += A[row][k] * B[l % N][k];
                    p->c[v] = s;
                }
            }
        },
        p);
    return p.c;
}

// Buffers with bounds: a dword at or past the range reads 0.
struct Resource {
    const uint8_t* base;
    uint32_t bytes;
};
template <typename V>
inline V buffer_load(Resource r, uint32_t at, uint32_t skip) {
    uint32_t d[sizeof(V) < 4 ? 1 : sizeof(V) / 4] = {};
    const uint64_t o = static_cast<uint64_t>(at) + skip;
    constexpr size_t step = sizeof(V) < 4 ? sizeof(V) : 4;
    for (size_t i = 0; i < sizeof(V); i += step)
        if (o + i + step <= r.bytes) std::memcpy(reinterpret_cast<uint8_t*>(d) + i, r.base + o + i, step);
    V v;
    std::memcpy(&v, d, sizeof(V));
    return v;
}
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));

inline uint32_t perm(uint32_t a, uint32_t b, uint32_t sel) {
    const uint64_t both = static_cast<uint64_t>(a) << 32 | b;
    uint32_t r = 0;
    for (int i = 0; i < 4; ++i) {
        const uint32_t s = sel >> 8 * i & 0xff;
        if (s > 7) fail("byte selector");
        r |= static_cast<uint32_t>(both >> 8 * s & 0xff) << 8 * i;
    }
    return r;
}
inline float fmed3(float a, float b, float c) { return fmaxf(fminf(fmaxf(a, b), c), fminf(a, b)); }
inline int frexp_exp(float v) {
    int e = 0;
    if (v != 0.0f && isfinite(v)) frexpf(v, &e);
    return e;
}

}  // namespace host

#define threadIdx host::thread_idx
#define blockIdx host::block_idx
#define gridDim host::grid_dim
#define blockDim host::block_dim
#define hipLaunchKernelGGL(...) host::launch(__VA_ARGS__)
inline void __syncthreads() { host::wait_as(host::kBarrier); }
template <typename T>
inline T atomicAdd(T* p, T v) {
    const T was = *p;
    *p = was + v;
    return was;
}
inline int __popcll(uint64_t v) { return __builtin_popcountll(v); }
inline uint32_t __umul24(uint32_t a, uint32_t b) { return (a & 0xffffff) * (b & 0xffffff); }
inline uint32_t __float_as_uint(float v) { return __builtin_bit_cast(uint32_t, v); }
inline float __uint_as_float(uint32_t v) { return __builtin_bit_cast(float, v); }
inline uint32_t __shfl_xor(uint32_t v, int mask, int) { return static_cast<uint32_t>(host::from_lane(v, host::lane_id() ^ mask)); }

#define __amdgpu_buffer_rsrc_t host::Resource
#define __builtin_amdgcn_make_buffer_rsrc(p, stride, n, flags) (host::Resource{static_cast<const uint8_t*>(p), static_cast<uint32_t>(n)})
#define __builtin_amdgcn_raw_buffer_load_b128(r, at, skip, aux) host::buffer_load<host::u4>(r, at, skip)
#define __builtin_amdgcn_raw_buffer_load_b64(r, at, skip, aux) host::buffer_load<host::u2>(r, at, skip)
#define __builtin_amdgcn_raw_buffer_load_b32(r, at, skip, aux) host::buffer_load<uint32_t>(r, at, skip)
#define __builtin_amdgcn_raw_buffer_load_b16(r, at, skip, aux) host::buffer_load<uint16_t>(r, at, skip)
#define __builtin_amdgcn_ballot_w64(...) host::ballot(__VA_ARGS__)
#define __builtin_amdgcn_readfirstlane(v) host::readfirstlane(v)
#define __builtin_amdgcn_readlane(v, l) static_cast<int>(host::from_lane(static_cast<uint32_t>(v), l))
#define __builtin_amdgcn_ds_bpermute(at, v) static_cast<int>(host::from_lane(static_cast<uint32_t>(v), (at) / 4))
#define __builtin_amdgcn_update_dpp(...) host::update_dpp(__VA_ARGS__)
#define __builtin_amdgcn_permlane16_swap(a, b, x, y) host::swap_rows<16>(a, b)
#define __builtin_amdgcn_permlane32_swap(a, b, x, y) host::swap_rows<32>(a, b)
#define __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, x, y, z) host::product<16, host::float4_t, 4>(a, b, c)
#define __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, x, y, z) host::product<32, host::float16_t, 16>(a, b, c)
#define __builtin_amdgcn_perm(a, b, s) host::perm(a, b, s)
#define __builtin_amdgcn_fmed3f(a, b, c) host::fmed3(a, b, c)
#define __builtin_amdgcn_exp2f(v) exp2f(v)
#define __builtin_amdgcn_rsq(v) (1.0 / sqrt(v))
#define __builtin_amdgcn_frexp_expf(v) host::frexp_exp(v)
#define __builtin_amdgcn_ubfe(v, at, n) ((v) >> (at) & ((1u << (n)) - 1))
#define __builtin_amdgcn_fdot2(a, b, c, d) (static_cast<float>((a)[0]) * static_cast<float>((b)[0]) + static_cast<float>((a)[1]) * static_cast<float>((b)[1]) + (c))
#define __builtin_amdgcn_fence(...)
// LDS written by some lanes of a wave and read by others: here each has to have come this far
#define __builtin_amdgcn_wave_barrier() static_cast<void>(host::ballot(true))
