// TEST INFRASTRUCTURE ONLY -- a tiny single-process SIMT emulator that lets the
// UNMODIFIED HIP sources in deft_amd/csrc be compiled for the host (clang++,
// -I tests/hipemu shadows <hip/hip_runtime.h>) and executed on CPU pointers, so
// kernel indexing / MFMA fragment logic can be unit-tested in the GPU-less build
// container.  It is NOT a fallback: the product loader (deft_amd/hiplib.py) only
// ever loads libdeft_hip.so built by hipcc for gfx950; this header is reachable
// from tests/ alone (tests/hipemu/build_emu.sh -> tests/hipemu/_build/libdeft_emu.so).
//
// Model: one fiber per GPU thread (hand-written x86-64 stack switch; ucontext elsewhere); the blocks of a launch
// are handed out to a persistent pool of OS threads (HIPEMU_THREADS, default = min(8, cores)), each running whole
// blocks one after another -- all emulator state, `__shared__` and dynamic LDS are thread_local, global atomics
// are real atomics.
// Wave-level collectives (MFMA, shuffles) rendezvous the 64 lanes of a wave;
// __syncthreads() rendezvous the block.  MFMA lane<->element maps follow
// /opt/skills/guides/cdna_hip_programming.md §3 (gfx950):
//   32x32x2 f32 : A[i=l&31][k=l>>5], B[k=l>>5][j=l&31],
//                 D reg r -> row=(r&3)+8*(r>>2)+4*(l>>5), col=l&31
//   16x16x4 f32 : A[l&15][k=l>>4],  B[k=l>>4][l&15], D reg r -> row=(l>>4)*4+r, col=l&15
// and accumulate as a k-ordered fmaf chain (bit-exact with the hardware).
#pragma once
#include <ucontext.h>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <atomic>
#include <condition_variable>
#include <functional>
#include <mutex>
#include <thread>
#include <vector>

// marks this build for the loader: its "device" pointers are host pointers (deft_amd/hiplib.py refuses to run the
// real library on CPU tensors, and this build on GPU tensors)
extern "C" __attribute__((weak, visibility("default"))) int deft_host_pointers(void) { return 1; }

#define __global__
#define __device__
#define __host__
#define __forceinline__ inline __attribute__((always_inline))
#define __shared__ static thread_local
#define __launch_bounds__(...)

struct dim3 {
    unsigned x, y, z;
    dim3(unsigned x_ = 1, unsigned y_ = 1, unsigned z_ = 1) : x(x_), y(y_), z(z_) {}
};
struct float2 { float x, y; };
struct alignas(16) float4 { float x, y, z, w; };
struct alignas(16) int4 { int x, y, z, w; };
struct int2 { int x, y; };
static inline float4 make_float4(float x, float y, float z, float w) { return float4{x, y, z, w}; }
static inline float2 make_float2(float x, float y) { return float2{x, y}; }
static inline int4 make_int4(int x, int y, int z, int w) { return int4{x, y, z, w}; }

typedef void* hipStream_t;
typedef int hipError_t;
#define hipSuccess 0
static inline hipError_t hipGetLastError() { return 0; }
static inline hipError_t hipPeekAtLastError() { return 0; }
static inline const char* hipGetErrorString(hipError_t) { return "emu"; }
static inline hipError_t hipMemsetAsync(void* p, int v, size_t n, hipStream_t) { memset(p, v, n); return 0; }
static inline hipError_t hipStreamSynchronize(hipStream_t) { return 0; }
enum { hipFuncAttributeMaxDynamicSharedMemorySize = 8 };
static inline hipError_t hipFuncSetAttribute(const void*, int, int) { return 0; }
namespace hipemu { inline void* dyn_lds() { alignas(16) static thread_local char buf[160 * 1024]; return buf; } }
#define DEFT_DYN_LDS(type, var) type* var = (type*)hipemu::dyn_lds()

// Fiber switch.  ucontext's swapcontext saves/restores the signal mask with two system calls per switch, which
// dominated the emulator's run time; on x86-64 a fiber switch here is six pushes, a stack-pointer swap and six pops.
#if defined(__x86_64__)
#define HIPEMU_ASM_SWITCH 1
extern "C" void hipemu_switch(void** save_sp, void* load_sp);
__asm__(".text\n.weak hipemu_switch\n.type hipemu_switch,@function\nhipemu_switch:\n"
        "  pushq %rbp\n  pushq %rbx\n  pushq %r12\n  pushq %r13\n  pushq %r14\n  pushq %r15\n"
        "  movq %rsp, (%rdi)\n  movq %rsi, %rsp\n"
        "  popq %r15\n  popq %r14\n  popq %r13\n  popq %r12\n  popq %rbx\n  popq %rbp\n  ret\n"
        ".size hipemu_switch, .-hipemu_switch\n");
#endif

namespace hipemu {
enum Yield { Y_NONE = 0, Y_WAVE = 1, Y_BLOCK = 2, Y_DONE = 3 };
struct State {
    dim3 tid, bid, bdim, gdim;
    int lane = 0, wave = 0;
#ifdef HIPEMU_ASM_SWITCH
    void* sched_sp = nullptr;
    void** cur_sp = nullptr;
#else
    ucontext_t sched, *cur = nullptr;
#endif
    int yield_code = 0;
    // wave exchange buffers: [parity][slot][lane]
    float xf[2][16][64];
    int parity = 0;
    // LDS-DMA pieces issued but not yet delivered ("late" mode, see dma_wait): one FIFO per thread of the block
    struct Pending { void* dst; unsigned char data[16]; };
    std::vector<std::vector<Pending>> dmaq;
    int cur_t = 0;
};
inline State& S() { static thread_local State s; return s; }
inline void yield(int code) {
    State& s = S();
    s.yield_code = code;
#ifdef HIPEMU_ASM_SWITCH
    hipemu_switch(s.cur_sp, s.sched_sp);
#else
    swapcontext(s.cur, &s.sched);
#endif
}
struct Fiber {
#ifdef HIPEMU_ASM_SWITCH
    void* sp = nullptr;
#else
    ucontext_t ctx;
#endif
    std::vector<char> stack;
    int state = Y_NONE;
};
inline std::function<void()>& body() { static thread_local std::function<void()> f; return f; }
// "Late DMA" mode: an LDS-DMA piece is delivered only when its wave WAITS for it (DEFT_WAIT_VM / DEFT_PIPE_BARRIER /
// __syncthreads -- the latest moment the hardware allows), not at issue (the earliest).  A kernel that reads a DMA stage
// before the issuing wave's vmcnt wait + a barrier then reads stale LDS here too; a piece still pending when its wave exits
// is reported (on the hardware it would land in LDS that may already belong to another workgroup).
inline int& late_dma() { static int on = 0; return on; }
inline void dma_wait(size_t keep) {
    State& s = S();
    if (s.dmaq.empty()) return;
    std::vector<State::Pending>& q = s.dmaq[s.cur_t];
    if (q.size() <= keep) return;
    const size_t n = q.size() - keep;
    for (size_t i = 0; i < n; ++i) memcpy(q[i].dst, q[i].data, 16);
    q.erase(q.begin(), q.begin() + n);
}
inline void trampoline() {
    body()();
    State& s = S();
    if (!s.dmaq.empty() && !s.dmaq[s.cur_t].empty()) {
        fprintf(stderr, "hipemu: thread %d exits with %zu LDS-DMA pieces in flight\n", s.cur_t, s.dmaq[s.cur_t].size());
        abort();
    }
    for (;;) yield(Y_DONE);          // a finished fiber is never resumed; never return into the fabricated frame
}

inline void run_block(const std::function<void()>& fn, dim3 grid, dim3 block, dim3 bid) {
    State& s = S();
    const int nthr = block.x * block.y * block.z;
    static thread_local std::vector<Fiber> fibers;
    if ((int)fibers.size() < nthr) fibers.resize(nthr);
    body() = fn;
    for (int t = 0; t < nthr; ++t) {
        Fiber& f = fibers[t];
        if (f.stack.empty()) f.stack.resize(256 * 1024);
#ifdef HIPEMU_ASM_SWITCH
        // fabricated frame: six callee-saved registers (zero) below the return address = trampoline; the slot of the
        // return address is 16-byte aligned, so the trampoline starts with the stack as after a call
        uintptr_t top = ((uintptr_t)(f.stack.data() + f.stack.size()) & ~(uintptr_t)15) - 16;
        void** frame = (void**)top;
        frame[0] = (void*)(void (*)())trampoline;
        for (int r = 1; r <= 6; ++r) frame[-r] = nullptr;
        f.sp = (void*)(frame - 6);
#else
        getcontext(&f.ctx);
        f.ctx.uc_stack.ss_sp = f.stack.data();
        f.ctx.uc_stack.ss_size = f.stack.size();
        f.ctx.uc_link = nullptr;
        makecontext(&f.ctx, (void (*)())trampoline, 0);
#endif
        f.state = Y_NONE;
    }
    const int nwave = (nthr + 63) / 64;
    std::vector<int> wparity(nwave, 0);
    if (late_dma()) { s.dmaq.resize(nthr); for (auto& q : s.dmaq) q.clear(); } else s.dmaq.clear();
    auto resume = [&](int t) {
        Fiber& f = fibers[t];
        s.cur_t = t;
        s.tid = dim3(t % block.x, (t / block.x) % block.y, t / (block.x * block.y));
        s.bid = bid; s.bdim = block; s.gdim = grid;
        s.lane = t & 63; s.wave = t >> 6;
        s.parity = wparity[t >> 6];
#ifdef HIPEMU_ASM_SWITCH
        s.cur_sp = &f.sp;
        hipemu_switch(&s.sched_sp, f.sp);
#else
        s.cur = &f.ctx;
        swapcontext(&s.sched, &f.ctx);
#endif
        f.state = s.yield_code;
    };
    for (;;) {
        int done = 0;
        for (int w = 0; w < nwave; ++w) {
            const int t0 = w * 64, t1 = (t0 + 64 < nthr) ? t0 + 64 : nthr;
            for (;;) {
                for (int t = t0; t < t1; ++t)
                    if (fibers[t].state == Y_NONE) resume(t);
                int nw = 0, nb = 0, nd = 0;
                for (int t = t0; t < t1; ++t) {
                    nw += fibers[t].state == Y_WAVE;
                    nb += fibers[t].state == Y_BLOCK;
                    nd += fibers[t].state == Y_DONE;
                }
                if (nw == t1 - t0) {            // whole wave at a wave collective -> release
                    wparity[w] ^= 1;
                    for (int t = t0; t < t1; ++t) fibers[t].state = Y_NONE;
                    continue;
                }
                if (nw != 0) {
                    fprintf(stderr, "hipemu: divergent wave collective (wave %d: %d at op, %d at barrier, %d done)\n", w, nw, nb, nd);
                    abort();
                }
                break;                          // all lanes at block barrier or done
            }
        }
        int nb = 0;
        for (int t = 0; t < nthr; ++t) { nb += fibers[t].state == Y_BLOCK; done += fibers[t].state == Y_DONE; }
        if (done == nthr) return;
        if (nb + done != nthr) { fprintf(stderr, "hipemu: scheduler stuck\n"); abort(); }
        for (int t = 0; t < nthr; ++t)
            if (fibers[t].state == Y_BLOCK) fibers[t].state = Y_NONE;
    }
}

inline int worker_count() {
    static const int n = [] {
        const char* e = getenv("HIPEMU_THREADS");
        int v = e ? atoi(e) : (int)std::thread::hardware_concurrency();
        return v < 1 ? 1 : (v > 8 ? 8 : v);
    }();
    return n;
}

// Worker threads live for the whole process: their thread_local fiber stacks (512 x 256 KB each) are then allocated
// and faulted in once, not once per launch.
struct Pool {
    std::vector<std::thread> th;
    std::mutex m;
    std::condition_variable cv, done_cv;
    const std::function<void()>* job = nullptr;
    long long gen = 0;
    int pending = 0;
    bool stop = false;
    explicit Pool(int n) {
        for (int i = 0; i < n; ++i) th.emplace_back([this] {
            long long seen = 0;
            for (;;) {
                const std::function<void()>* j;
                {
                    std::unique_lock<std::mutex> lk(m);
                    cv.wait(lk, [&] { return stop || gen != seen; });
                    if (stop) return;
                    seen = gen; j = job;
                }
                (*j)();
                std::lock_guard<std::mutex> lk(m);
                if (--pending == 0) done_cv.notify_one();
            }
        });
    }
    ~Pool() {
        { std::lock_guard<std::mutex> lk(m); stop = true; }
        cv.notify_all();
        for (auto& t : th) t.join();
    }
    void run(const std::function<void()>& work) {
        { std::lock_guard<std::mutex> lk(m); job = &work; pending = (int)th.size(); ++gen; }
        cv.notify_all();
        work();
        std::unique_lock<std::mutex> lk(m);
        done_cv.wait(lk, [&] { return pending == 0; });
    }
};
inline Pool& pool() { static Pool p(worker_count() - 1); return p; }

template <typename F>
inline void launch(F&& fn, dim3 grid, dim3 block) {
    const long long total = (long long)grid.x * grid.y * grid.z;
    const std::function<void()> f = fn;
    std::atomic<long long> next{0};
    const std::function<void()> work = [&]() {
        for (long long b = next.fetch_add(1); b < total; b = next.fetch_add(1))
            run_block(f, grid, block, dim3((unsigned)(b % grid.x), (unsigned)((b / grid.x) % grid.y), (unsigned)(b / ((long long)grid.x * grid.y))));
    };
    if (total < 4 || worker_count() <= 1) { work(); return; }
    pool().run(work);
}

// wave exchange: deposit up to two floats, rendezvous, then read any lane's deposit
inline void exchange(float a, float b, const float*& ra, const float*& rb) {
    State& s = S();
    const int p = s.parity ^ 1;               // buffer for THIS op (parity flips on release)
    const int lane = s.lane;
    s.xf[p][0][lane] = a;
    s.xf[p][1][lane] = b;
    yield(Y_WAVE);
    ra = S().xf[p][0];
    rb = S().xf[p][1];
}
}  // namespace hipemu

#define threadIdx (hipemu::S().tid)
#define blockIdx (hipemu::S().bid)
#define blockDim (hipemu::S().bdim)
#define gridDim (hipemu::S().gdim)
static const int warpSize = 64;

#define hipLaunchKernelGGL(kernel, grid, block, shmem, stream, ...) \
    hipemu::launch([=]() { kernel(__VA_ARGS__); }, dim3(grid), dim3(block))

// (hipcc's __syncthreads() is fence + s_barrier: it drains vmcnt when LDS-DMA pieces are outstanding)
static inline void __syncthreads() { hipemu::dma_wait(0); hipemu::yield(hipemu::Y_BLOCK); }

typedef float __attribute__((ext_vector_type(16))) hipemu_f32x16;
typedef float __attribute__((ext_vector_type(4))) hipemu_f32x4;

static inline hipemu_f32x16 __builtin_amdgcn_mfma_f32_32x32x2f32(float a, float b, hipemu_f32x16 c, int, int, int) {
    const float *A, *B;
    const int lane = hipemu::S().lane;
    hipemu::exchange(a, b, A, B);
    const int col = lane & 31, hi = lane >> 5;
    for (int r = 0; r < 16; ++r) {
        const int row = (r & 3) + 8 * (r >> 2) + 4 * hi;
        float acc = c[r];
        for (int k = 0; k < 2; ++k) acc = fmaf(A[row + 32 * k], B[col + 32 * k], acc);
        c[r] = acc;
    }
    return c;
}
// 32x32x16 bf16 (gfx950): lane l feeds row/col l&31 with the 8 consecutive k of group l>>5; C/D as 32x32x2.
// Products of bf16 values are exact in fp32; the hardware's internal summation order is not specified, here k-ordered.
typedef __bf16 hipemu_bf16x8 __attribute__((ext_vector_type(8)));
static inline hipemu_f32x16 __builtin_amdgcn_mfma_f32_32x32x16_bf16(hipemu_bf16x8 a, hipemu_bf16x8 b, hipemu_f32x16 c, int, int, int) {
    hipemu::State& s = hipemu::S();
    const int p = s.parity ^ 1, lane = s.lane;
    for (int e = 0; e < 8; ++e) { s.xf[p][e][lane] = (float)a[e]; s.xf[p][8 + e][lane] = (float)b[e]; }
    hipemu::yield(hipemu::Y_WAVE);
    hipemu::State& t = hipemu::S();
    const int col = lane & 31, hi = lane >> 5;
    for (int r = 0; r < 16; ++r) {
        const int row = (r & 3) + 8 * (r >> 2) + 4 * hi;
        float acc = c[r];
        for (int kg = 0; kg < 2; ++kg)
            for (int e = 0; e < 8; ++e) acc = fmaf(t.xf[p][e][row + 32 * kg], t.xf[p][8 + e][col + 32 * kg], acc);
        c[r] = acc;
    }
    return c;
}
// 32x32x16 f16 (gfx950): same fragment layout; products of fp16 values (11 x 11 significant bits) are exact in fp32 too.
typedef _Float16 hipemu_f16x8 __attribute__((ext_vector_type(8)));
static inline hipemu_f32x16 __builtin_amdgcn_mfma_f32_32x32x16_f16(hipemu_f16x8 a, hipemu_f16x8 b, hipemu_f32x16 c, int, int, int) {
    hipemu::State& s = hipemu::S();
    const int p = s.parity ^ 1, lane = s.lane;
    for (int e = 0; e < 8; ++e) { s.xf[p][e][lane] = (float)a[e]; s.xf[p][8 + e][lane] = (float)b[e]; }
    hipemu::yield(hipemu::Y_WAVE);
    hipemu::State& t = hipemu::S();
    const int col = lane & 31, hi = lane >> 5;
    for (int r = 0; r < 16; ++r) {
        const int row = (r & 3) + 8 * (r >> 2) + 4 * hi;
        float acc = c[r];
        for (int kg = 0; kg < 2; ++kg)
            for (int e = 0; e < 8; ++e) acc = fmaf(t.xf[p][e][row + 32 * kg], t.xf[p][8 + e][col + 32 * kg], acc);
        c[r] = acc;
    }
    return c;
}
// 16x16x32 bf16 (gfx950): lane l feeds row/col l&15 with the 8 consecutive k of group l>>4; D reg r of lane l is row 4*(l>>4)+r, col l&15.
static inline hipemu_f32x4 __builtin_amdgcn_mfma_f32_16x16x32_bf16(hipemu_bf16x8 a, hipemu_bf16x8 b, hipemu_f32x4 c, int, int, int) {
    hipemu::State& s = hipemu::S();
    const int p = s.parity ^ 1, lane = s.lane;
    for (int e = 0; e < 8; ++e) { s.xf[p][e][lane] = (float)a[e]; s.xf[p][8 + e][lane] = (float)b[e]; }
    hipemu::yield(hipemu::Y_WAVE);
    hipemu::State& t = hipemu::S();
    const int col = lane & 15, q = lane >> 4;
    for (int r = 0; r < 4; ++r) {
        const int row = q * 4 + r;
        float acc = c[r];
        for (int kg = 0; kg < 4; ++kg)
            for (int e = 0; e < 8; ++e) acc = fmaf(t.xf[p][e][row + 16 * kg], t.xf[p][8 + e][col + 16 * kg], acc);
        c[r] = acc;
    }
    return c;
}
// 16x16x32 f16 (gfx950): the same fragment layout on fp16 inputs
static inline hipemu_f32x4 __builtin_amdgcn_mfma_f32_16x16x32_f16(hipemu_f16x8 a, hipemu_f16x8 b, hipemu_f32x4 c, int, int, int) {
    hipemu::State& s = hipemu::S();
    const int p = s.parity ^ 1, lane = s.lane;
    for (int e = 0; e < 8; ++e) { s.xf[p][e][lane] = (float)a[e]; s.xf[p][8 + e][lane] = (float)b[e]; }
    hipemu::yield(hipemu::Y_WAVE);
    hipemu::State& t = hipemu::S();
    const int col = lane & 15, q = lane >> 4;
    for (int r = 0; r < 4; ++r) {
        const int row = q * 4 + r;
        float acc = c[r];
        for (int kg = 0; kg < 4; ++kg)
            for (int e = 0; e < 8; ++e) acc = fmaf(t.xf[p][e][row + 16 * kg], t.xf[p][8 + e][col + 16 * kg], acc);
        c[r] = acc;
    }
    return c;
}
static inline hipemu_f32x4 __builtin_amdgcn_mfma_f32_16x16x4f32(float a, float b, hipemu_f32x4 c, int, int, int) {
    const float *A, *B;
    const int lane = hipemu::S().lane;
    hipemu::exchange(a, b, A, B);
    const int col = lane & 15, q = lane >> 4;
    for (int r = 0; r < 4; ++r) {
        const int row = q * 4 + r;
        float acc = c[r];
        for (int k = 0; k < 4; ++k) acc = fmaf(A[row + 16 * k], B[col + 16 * k], acc);
        c[r] = acc;
    }
    return c;
}
static inline float __shfl_xor(float v, int mask, int = 64) {
    const float *A, *B; const int lane = hipemu::S().lane;
    hipemu::exchange(v, 0.f, A, B);
    return A[(lane ^ mask) & 63];
}
static inline float __shfl_down(float v, int d, int = 64) {
    const float *A, *B; const int lane = hipemu::S().lane;
    hipemu::exchange(v, 0.f, A, B);
    return A[lane + d < 64 ? lane + d : lane];
}
static inline float __shfl(float v, int src, int = 64) {
    const float *A, *B;
    hipemu::exchange(v, 0.f, A, B);
    return A[src & 63];
}
static inline int __shfl_xor(int v, int mask, int = 64) {
    float f; memcpy(&f, &v, 4); f = __shfl_xor(f, mask); memcpy(&v, &f, 4); return v;
}
static inline int __shfl_down(int v, int d, int = 64) {
    float f; memcpy(&f, &v, 4); f = __shfl_down(f, d); memcpy(&v, &f, 4); return v;
}
static inline int __shfl(int v, int src, int = 64) {
    float f; memcpy(&f, &v, 4); f = __shfl(f, src); memcpy(&v, &f, 4); return v;
}
static inline unsigned __shfl_xor(unsigned v, int mask, int = 64) { return (unsigned)__shfl_xor((int)v, mask); }
static inline unsigned __shfl_down(unsigned v, int d, int = 64) { return (unsigned)__shfl_down((int)v, d); }

template <typename T> static inline T atomicAdd(T* p, T v) {
    T o = __atomic_load_n(p, __ATOMIC_RELAXED);
    while (!__atomic_compare_exchange_n(p, &o, (T)(o + v), true, __ATOMIC_RELAXED, __ATOMIC_RELAXED)) {}
    return o;
}
static inline float atomicAdd(float* p, float v) {
    unsigned* q = (unsigned*)p;
    unsigned o = __atomic_load_n(q, __ATOMIC_RELAXED), n;
    float f;
    do { memcpy(&f, &o, 4); f += v; memcpy(&n, &f, 4); } while (!__atomic_compare_exchange_n(q, &o, n, true, __ATOMIC_RELAXED, __ATOMIC_RELAXED));
    memcpy(&f, &o, 4);
    return f;
}
template <typename T> static inline T atomicMax(T* p, T v) {
    T o = __atomic_load_n(p, __ATOMIC_RELAXED);
    while (v > o && !__atomic_compare_exchange_n(p, &o, v, true, __ATOMIC_RELAXED, __ATOMIC_RELAXED)) {}
    return o;
}
static inline void __threadfence() { __atomic_thread_fence(__ATOMIC_SEQ_CST); }
// split-K hand-over hooks of deft_amd/csrc/common.h (blocks run on several OS threads here)
#define DEFT_WS_HOOKS 1
static inline void deft_ws_store(float* p, float v) { __atomic_store((unsigned*)p, (unsigned*)&v, __ATOMIC_RELAXED); }
static inline float deft_ws_load(const float* p) { float v; __atomic_load((const unsigned*)p, (unsigned*)&v, __ATOMIC_RELAXED); return v; }
static inline void deft_ws_publish() { __atomic_thread_fence(__ATOMIC_SEQ_CST); }
static inline int deft_ws_ticket(int* p) { return __atomic_fetch_add(p, 1, __ATOMIC_SEQ_CST); }
static inline void deft_ws_reset(int* p) { __atomic_store_n(p, 0, __ATOMIC_SEQ_CST); }
static inline float __fdividef(float a, float b) { return a / b; }
static inline float __frcp_rn(float a) { return 1.0f / a; }
static inline int __float_as_int(float f) { int i; memcpy(&i, &f, 4); return i; }
static inline unsigned __float_as_uint(float f) { unsigned i; memcpy(&i, &f, 4); return i; }
static inline float __int_as_float(int i) { float f; memcpy(&f, &i, 4); return f; }
static inline float __uint_as_float(unsigned i) { float f; memcpy(&f, &i, 4); return f; }
static inline void __builtin_amdgcn_s_setprio(int) {}
// buffer-load hooks of deft_amd/csrc/common.h: num_records = 2^31-1, offsets >= 2^31 read as zero
#define DEFT_BUFFER_HOOKS 1
struct deft_rsrc_t { const char* base; unsigned n; };
static inline deft_rsrc_t deft_make_rsrc(const void* base) { return deft_rsrc_t{(const char*)base, 0x7FFFFFFFu}; }
static inline hipemu_f32x4 deft_buffer_load_x4(deft_rsrc_t r, unsigned byte_off) {
    hipemu_f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (byte_off < r.n && byte_off + 16u <= r.n) memcpy(&v, r.base + byte_off, 16);
    return v;
}
static inline void hipemu_dma_deposit(void* dst, const hipemu_f32x4& v) {
    hipemu::State& s = hipemu::S();
    if (s.dmaq.empty()) { memcpy(dst, &v, 16); return; }          // default: delivered at issue
    hipemu::State::Pending p; p.dst = dst; memcpy(p.data, &v, 16);
    s.dmaq[s.cur_t].push_back(p);
}
static inline void deft_buffer_load_lds_x4(deft_rsrc_t r, float* lds_wave_base, unsigned byte_off) {
    const hipemu_f32x4 v = deft_buffer_load_x4(r, byte_off);
    hipemu_dma_deposit(lds_wave_base + 4 * hipemu::S().lane, v);
}
static inline void deft_buffer_load_lds_x4s(deft_rsrc_t r, void* lds_wave_base, unsigned voff, unsigned soff) {
    hipemu_f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (voff < r.n && voff + 16u <= r.n) memcpy(&v, r.base + voff + soff, 16);      // range check on voff alone, like the hardware
    hipemu_dma_deposit((char*)lds_wave_base + 16 * hipemu::S().lane, v);
}
// the raw barrier does not wait for DMA pieces; the vmcnt forms deliver all but the newest N of the calling thread's wave
#define DEFT_PIPE_BARRIER(N) do { hipemu::dma_wait(N); hipemu::yield(hipemu::Y_BLOCK); } while (0)
#define DEFT_PIPE_BARRIER_ONLY() hipemu::yield(hipemu::Y_BLOCK)
#define DEFT_WAIT_VM(N) hipemu::dma_wait(N)
// (the lanes of a wave run one after another here: meet before another lane's pieces are read, or overwritten)
#define DEFT_WAVE_VM(N) do { hipemu::dma_wait(N); hipemu::yield(hipemu::Y_WAVE); } while (0)
#define DEFT_WAVE_LGKM() hipemu::yield(hipemu::Y_WAVE)
// hooks of deft_amd/csrc/attn.hip: the transposing 16-bit LDS read (lane i of a group of 16 gets column i of the 4 x 16 block whose row (j >> 2),
// 4-element chunk (j & 3) lane j addresses), ballot, base-2 exponential and logarithm
#define DEFT_LDS_TR_HOOK 1
typedef short hipemu_s16x4 __attribute__((ext_vector_type(4)));
static inline hipemu_s16x4 deft_lds_read_tr16(const void* ptr) {
    hipemu::State& s = hipemu::S();
    const int p = s.parity ^ 1, lane = s.lane;
    short v[4];
    memcpy(v, ptr, 8);
    for (int e = 0; e < 4; ++e) s.xf[p][e][lane] = (float)v[e];
    hipemu::yield(hipemu::Y_WAVE);
    hipemu::State& t = hipemu::S();
    const int g = lane & ~15, i = lane & 15;
    hipemu_s16x4 r;
    for (int e = 0; e < 4; ++e) r[e] = (short)t.xf[p][i & 3][g + 4 * e + (i >> 2)];
    return r;
}
typedef deft_rsrc_t lds_src;
typedef char* lds_at;
static inline lds_at lds_address(char* lds) { return lds; }
static inline lds_src lds_source(const char* base, unsigned bytes) { return lds_src{base, bytes}; }
static inline void lds_fetch(const lds_src& s, lds_at lds, unsigned off) { deft_buffer_load_lds_x4(s, (float*)lds, off); }
static inline unsigned long long deft_ballot(bool b) {
    const float *A, *B;
    hipemu::exchange(b ? 1.f : 0.f, 0.f, A, B);
    unsigned long long m = 0;
    for (int l = 0; l < 64; ++l) m |= (unsigned long long)(A[l] != 0.f) << l;
    return m;
}
// hooks of deft_amd/csrc/rotary.hip
#define DEFT_DPP_HOOK 1
template <int S> static inline float deft_add_xor(float v) { return v + __shfl_xor(v, S); }
static inline float deft_rsq(float x) { return 1.f / sqrtf(x); }
static inline float deft_exp2(float x) { return exp2f(x); }
static inline float deft_log2(float x) { return log2f(x); }
static inline unsigned __umulhi(unsigned a, unsigned b) { return (unsigned)(((unsigned long long)a * b) >> 32); }
static inline int __popcll(unsigned long long x) { return __builtin_popcountll(x); }
extern "C" __attribute__((weak, visibility("default"))) void hipemu_set_late_dma(int on) { hipemu::late_dma() = on; }
#define DEFT_OPAQUE(v) ((void)(v))
#define DEFT_OPAQUE_NV(v) ((void)(v))
// the two-fp16-piece split of a pair of values (csrc/common.h: v_cvt_pk_f16_f32 + v_fma_mix{lo,hi}_f16 on the device), as the C++ expression
#define DEFT_F16_SPLIT_HOOK 1
static inline void deft_split2_pair_scaled(float x0, float x1, float sc, unsigned& h, unsigned& m) {
    const float y0 = x0 * sc, y1 = x1 * sc;                        // (sc is a power of two: exact)
    const _Float16 h0 = (_Float16)y0, h1 = (_Float16)y1;
    const _Float16 m0 = (_Float16)(y0 - (float)h0), m1 = (_Float16)(y1 - (float)h1);
    unsigned short b[4];
    __builtin_memcpy(&b[0], &h0, 2); __builtin_memcpy(&b[1], &h1, 2); __builtin_memcpy(&b[2], &m0, 2); __builtin_memcpy(&b[3], &m1, 2);
    h = (unsigned)b[0] | ((unsigned)b[1] << 16);
    m = (unsigned)b[2] | ((unsigned)b[3] << 16);
}
static inline void deft_split2_pair(float x0, float x1, unsigned& h, unsigned& m) { deft_split2_pair_scaled(x0, x1, 1.f, h, m); }
#define DEFT_FAST_RCP(x) (1.0f / (x))
#define DEFT_RINT_HOOK 1
static inline int deft_rint(double v) { return (int)std::nearbyint(v); }
static inline void __builtin_amdgcn_sched_barrier(int) {}
static inline void __builtin_amdgcn_sched_group_barrier(int, int, int) {}
static inline int __builtin_amdgcn_readfirstlane(int v) { return v; }
