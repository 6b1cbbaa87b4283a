"""Where the rotary, cache and one-token attention kernels read and write: their source compiled for the CPU and run as a GPU runs it, a fiber a
thread, lanes meeting at every exchange, matrix product and barrier, over buffers that end at an unmapped page (planes, tables, rows, workspace, LDS).  An access past either
end ends the program with the case that made it, and the results are compared with plain sums.  No GPU."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "machx_inference_engine_amd", "csrc")

SHIM = r"""
#include <hip/hip_runtime.h>
#include <algorithm>
#include <functional>
#include <math.h>
#include <signal.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <sys/mman.h>
#include <type_traits>
#include <ucontext.h>
#include <unistd.h>
#include <vector>
#undef __global__
#undef __device__
#undef __host__
#undef __shared__
#undef __forceinline__
#undef __launch_bounds__
#define __global__
#define __device__
#define __host__
#define __shared__ static
#define __forceinline__ inline
#define __launch_bounds__(...)
template <class A, class B> static inline std::common_type_t<A, B> min(A a, B b) { return (std::common_type_t<A, B>)a < (std::common_type_t<A, B>)b ? a : b; }
template <class A, class B> static inline std::common_type_t<A, B> max(A a, B b) { return (std::common_type_t<A, B>)a < (std::common_type_t<A, B>)b ? b : a; }
struct Idx { uint32_t x, y, z; };
static Idx blockIdx, blockDim, gridDim;
static char* shim_lds;

// ---- a workgroup: one fiber a thread, resumed in turn; a fiber that waits for others goes to the back
struct Fiber { ucontext_t at; bool done; };
constexpr int kMost = 512, kStack = 192 * 1024;
static Fiber fiber[kMost];
static ucontext_t home;
static int now, threads;
static Idx threadIdx;
static char* stacks;
static long idle;
static void on_stuck();
static void yield() {
    if (++idle > 40l * kMost) on_stuck();
    const int me = now;
    swapcontext(&fiber[me].at, &home);
}
// threads of the group [first, first + size) meet: those that have ended do not count
struct Meet { int count = 0; long round = 0; };
static Meet meet[11][kMost];
static int living(int first, int size) { int n = 0; for (int i = first; i < first + size && i < threads; ++i) n += !fiber[i].done; return n; }
static void rendezvous(int kind, int size) {
    const int first = now / size * size;
    Meet& m = meet[kind][first];
    const long round = m.round;
    ++m.count;
    while (m.round == round) {
        if (m.count >= living(first, size)) { m.count = 0; ++m.round; idle = 0; return; }
        yield();
    }
}
static uint64_t slot[kMost][8];
template <class T> static T from_lane(T v, int kind, int size, int lane_of_group) {   // lane_of_group < 0: nobody's, zero
    static_assert(sizeof(T) <= 64, "");
    memcpy(slot[now], &v, sizeof v);
    rendezvous(kind, size);
    T r{};
    if (lane_of_group >= 0) memcpy(&r, slot[now / size * size + lane_of_group], sizeof r);
    rendezvous(kind, size);
    return r;
}
static void __syncthreads() { rendezvous(0, kMost); }
static int lane_id() { return now & 63; }
static int shim_dpp(int old, int v, int ctrl, int row_mask, int, bool bound) {
    const int l = lane_id(), row = l >> 4;
    if (ctrl == 0xB1) return from_lane(v, 1, 4, (l & 3) ^ 1);
    if (ctrl == 0x4E) return from_lane(v, 1, 4, (l & 3) ^ 2);
    if (ctrl == 0x141) return from_lane(v, 2, 8, 7 - (l & 7));
    if (ctrl == 0x140) return from_lane(v, 3, 16, 15 - (l & 15));
    int src = -1;
    if (ctrl > 0x110 && ctrl <= 0x11F) src = (l & 15) >= ctrl - 0x110 ? l - (ctrl - 0x110) : -1;
    else if (ctrl == 0x142) src = row > 0 ? row * 16 - 1 : -1;
    else if (ctrl == 0x143) src = row > 1 ? 31 : -1;
    else abort();
    const int got = from_lane(v, 4, 64, src);
    return (row_mask >> row & 1) && src >= 0 ? got : bound && (row_mask >> row & 1) ? 0 : old;
}
static uint64_t __ballot(bool v) {
    const uint64_t mine = v;
    memcpy(slot[now], &mine, 8);
    rendezvous(4, 64);
    uint64_t r = 0;
    for (int i = 0; i < 64; ++i) if (!fiber[now / 64 * 64 + i].done) r |= slot[now / 64 * 64 + i][0] << i;
    rendezvous(4, 64);
    return r;
}
static bool __any(bool v) { return __ballot(v) != 0; }
struct Two { uint32_t v[2]; uint32_t operator[](int i) const { return v[i]; } };
static Two shim_swap(uint32_t a, uint32_t b, int width) {   // halves (or rows) of one operand against the other's
    const uint32_t l = lane_id();
    const bool odd = l & width;
    const uint32_t other_a = from_lane(a, 5, 64, l ^ width), other_b = from_lane(b, 5, 64, l ^ width);
    return Two{{odd ? other_b : a, odd ? b : other_a}};
}
static uint32_t shim_perm(uint32_t hi, uint32_t lo, uint32_t sel) {
    uint32_t r = 0;
    for (int i = 0; i < 4; ++i) {
        const uint32_t s = sel >> (8 * i) & 0xFF;
        if (s > 7) abort();
        r |= ((s < 4 ? lo >> (8 * s) : hi >> (8 * (s - 4))) & 0xFF) << (8 * i);
    }
    return r;
}
typedef _Float16 shim_h8 __attribute__((ext_vector_type(8)));
typedef float shim_f4 __attribute__((ext_vector_type(4)));
static shim_h8 mfma_a[kMost], mfma_b[kMost];
static shim_f4 shim_mfma(shim_h8 a, shim_h8 b, shim_f4 c, int, int, int) {
    mfma_a[now] = a; mfma_b[now] = b;
    rendezvous(6, 64);
    const int w = now / 64 * 64, l = lane_id(), col = l & 15;
    for (int j = 0; j < 4; ++j) {
        const int row = (l >> 4) * 4 + j;
        double s = c[j];
        for (int k = 0; k < 32; ++k) s += (double)(float)mfma_a[w + k / 8 * 16 + row][k % 8] * (double)(float)mfma_b[w + k / 8 * 16 + col][k % 8];
        c[j] = (float)s;
    }
    rendezvous(6, 64);
    return c;
}
#define __builtin_amdgcn_update_dpp shim_dpp
#define __builtin_amdgcn_perm shim_perm
#define __builtin_amdgcn_mfma_f32_16x16x32_f16 shim_mfma
#define __builtin_amdgcn_permlane32_swap(a, b, c, d) shim_swap(a, b, 32)
#define __builtin_amdgcn_permlane16_swap(a, b, c, d) shim_swap(a, b, 16)
#define __builtin_amdgcn_readfirstlane(v) from_lane((v), 7, 64, 0)
#define __builtin_amdgcn_readlane(v, l) from_lane((v), 7, 64, (l))
#define __builtin_amdgcn_exp2f exp2f
#define __builtin_amdgcn_fence(a, b)
#define __builtin_amdgcn_wave_barrier() rendezvous(8, 64)
#define __builtin_amdgcn_sdot4(a, b, c, d) (c)
#define __popcll __builtin_popcountll
#define __ffsll __builtin_ffsll
"""

CHECK = r"""
using namespace mxq;
static char what[400];
static void say(const char* m) { if (write(1, m, strlen(m)) < 0) return; if (write(1, what, strlen(what)) < 0) return; }
static void on_fault(int) { say("access outside its buffer: "); _exit(3); }
static void on_stuck() { say("lanes wait for each other: "); _exit(4); }
static void wrong(const char* m) { say(m); _exit(5); }
// n bytes that end where an unmapped page starts; another one lies in front
struct Held {
    uint8_t* p; size_t n, up;
    Held(size_t bytes) : n(bytes), up((bytes + 4095) / 4096 * 4096) {
        uint8_t* m = static_cast<uint8_t*>(mmap(nullptr, up + 8192, PROT_NONE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0));
        mprotect(m + 4096, up, PROT_READ | PROT_WRITE);
        p = m + 4096 + up - n;
    }
    ~Held() { munmap(p + n - up - 4096, up + 8192); }
    template <class T> T* as() { return reinterpret_cast<T*>(p); }
};
static std::function<void()> body;
static void entry() { body(); fiber[now].done = true; idle = 0; swapcontext(&fiber[now].at, &home); }
template <class Fn> static void run(uint32_t n, uint32_t gx, uint32_t gy, size_t lds_bytes, Fn fn) {
    if (!stacks) stacks = static_cast<char*>(malloc((size_t)kMost * kStack));
    Held l(lds_bytes ? lds_bytes : 16);
    shim_lds = l.as<char>();
    blockDim = {n, 1, 1}; gridDim = {gx, gy, 1}; threads = n;
    body = fn;
    for (uint32_t y = 0; y < gy; ++y)
        for (uint32_t x = 0; x < gx; ++x) {
            blockIdx = {x, y, 0};
            memset(l.p, 0xFF, l.n);
            for (uint32_t t = 0; t < n; ++t) {
                fiber[t].done = false;
                getcontext(&fiber[t].at);
                fiber[t].at.uc_stack.ss_sp = stacks + (size_t)t * kStack;
                fiber[t].at.uc_stack.ss_size = kStack;
                fiber[t].at.uc_link = &home;
                makecontext(&fiber[t].at, entry, 0);
            }
            idle = 0;
            for (uint32_t left = n; left;)
                for (uint32_t t = 0; t < n; ++t) {
                    if (fiber[t].done) continue;
                    now = t;
                    threadIdx = {t, 0, 0};
                    swapcontext(&home, &fiber[t].at);
                    left -= fiber[t].done;
                }
        }
}
static uint32_t seed = 1;
static uint32_t rnd(uint32_t n) { seed = seed * 1664525u + 1013904223u; return (seed >> 8) % n; }
static float real() { return ((int)rnd(2001) - 1000) / 500.f; }
static void fill(half_t* p, size_t n) { for (size_t i = 0; i < n; ++i) p[i] = (half_t)real(); }
"""

ATTENTION = r"""
template <bool Q8, int DP, int NBLK, bool FULL> static void one(uint32_t D, uint32_t Hkv, uint32_t G, uint32_t ps, uint32_t window, uint32_t shares, std::vector<int32_t> lens) {
    const uint32_t B = (uint32_t)lens.size(), Hq = Hkv * G;
    uint32_t most = 1, pages = 0;
    for (int32_t n : lens) { const uint32_t need = n > 0 ? (n + ps - 1) / ps : 0; most = std::max(most, need); pages += need; }
    if (pages == 0) pages = 1;
    snprintf(what, sizeof what, "attention, %s D=%u Hkv=%u G=%u pages of %u, window %u, %u shares, %u sequences of %d..\n", Q8 ? "Q8_0" : "fp16", D, Hkv, G, ps, window, shares, B, lens[0]);
    const size_t values = (size_t)pages * Hkv * ps * D;
    Held q(2 * (size_t)B * Hq * D), k(values * (Q8 ? 1 : 2)), v(values * (Q8 ? 1 : 2)), kd(values / 16), vd(values / 16), table(4 * (size_t)B * most), len(4 * B), sinks(4 * Hq),
        out(2 * (size_t)B * Hq * D), q8((size_t)B * Hq * D / 32 * 40 + 8), ws((((size_t)shares + B) * Hq * (D + 2) * 4 + B * 8 + 15) / 16 * 16);   // it begins at a multiple of 16
    fill(q.as<half_t>(), (size_t)B * Hq * D);
    if (Q8) {
        for (size_t i = 0; i < values; ++i) { k.as<int8_t>()[i] = (int8_t)((int)rnd(255) - 127); v.as<int8_t>()[i] = (int8_t)((int)rnd(255) - 127); }
        for (size_t i = 0; i < values / 32; ++i) { kd.as<half_t>()[i] = (half_t)(0.002f + 0.00001f * rnd(999)); vd.as<half_t>()[i] = (half_t)(0.002f + 0.00001f * rnd(999)); }
    } else { fill(k.as<half_t>(), values); fill(v.as<half_t>(), values); }
    uint32_t next = pages;
    for (uint32_t b = 0; b < B; ++b) {
        len.as<int32_t>()[b] = lens[b];
        for (uint32_t i = 0; i < most; ++i) table.as<int32_t>()[b * most + i] = lens[b] > 0 && i < (lens[b] + ps - 1) / ps ? (int32_t)--next : 2147483647;
    }
    for (uint32_t h = 0; h < Hq; ++h) sinks.as<float>()[h] = real();
    memset(out.p, 0xFF, out.n);
    AttnArgs a = {};
    a.q = q.as<half_t>(); a.q_stride = (uint64_t)Hq * D; a.k = k.p; a.v = v.p; a.k_d = kd.as<half_t>(); a.v_d = vd.as<half_t>();
    a.table = table.as<int32_t>(); a.lens = len.as<int32_t>(); a.sinks = sinks.as<float>(); a.out = out.as<half_t>(); a.out_q8 = D % 32 ? nullptr : q8.p;
    a.part_o = ws.as<float>(); a.part_ml = a.part_o + ((size_t)shares + B) * Hq * D; a.parts = reinterpret_cast<uint32_t*>(a.part_ml + ((size_t)shares + B) * Hq * 2);
    a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.D = D; a.max_pages = most; a.n_pages = pages; a.page_size = ps; a.window = window; a.shares = shares;
    a.page_shift = (ps & (ps - 1)) == 0 ? (uint32_t)__builtin_ctz(ps) : 32u;
    a.scale = 0.3f * kLog2e;
    const uint32_t heads = std::min(G, 16u);
    const size_t keys = kWaves * kTile * (Q8 ? DP + 4 * NBLK : 2 * DP) + (DP > 128 ? DP * 32 : 0), sums = kWaves * (32 + heads * (DP + 4)) * 4;   // as the launch asks for
    run(kWaves * 64, shares ? shares : B, Hkv * ((G + 15) / 16), std::max(keys, sums), [&] { attn_decode_kernel<Q8, DP, NBLK, FULL>(a); });
    if (shares) {
        uint32_t groups = std::min((shares / B + 4) / 4, 512 / (D / 4));
        run((groups * (D / 4) + 63) / 64 * 64, B * Hq, 1, groups * D * 4, [&] { attn_join_kernel(a, groups); });
    }
    for (uint32_t b = 0; b < B; ++b)
        for (uint32_t h = 0; h < Hq; ++h) {
            const uint32_t n = lens[b] > 0 ? lens[b] : 0, lo = window && n > window ? n - window : 0, hk = h / G;
            std::vector<double> x, sum(D, 0.0);
            double top = sinks.as<float>()[h], total;
            auto at = [&](uint32_t t) { return (((size_t)table.as<int32_t>()[b * most + t / ps]) * Hkv + hk) * ps + t % ps; };
            auto value = [&](Held& p, Held& d, size_t row, uint32_t i) {
                return Q8 ? (double)p.as<int8_t>()[row * D + i] * (double)(float)d.as<half_t>()[(row * D + i) / 32] : (double)(float)p.as<half_t>()[row * D + i];
            };
            for (uint32_t t = lo; t < n; ++t) {
                double s = 0;
                for (uint32_t i = 0; i < D; ++i) s += (double)(float)q.as<half_t>()[((size_t)b * Hq + h) * D + i] * value(k, kd, at(t), i);
                x.push_back(0.3 * s);
                top = std::max(top, x.back());
            }
            total = exp(sinks.as<float>()[h] - top);
            for (uint32_t t = lo; t < n; ++t) {
                const double p = exp(x[t - lo] - top);
                total += p;
                for (uint32_t i = 0; i < D; ++i) sum[i] += p * value(v, vd, at(t), i);
            }
            for (uint32_t i = 0; i < D; ++i) {
                const double want = n ? sum[i] / total : 0.0, got = (double)(float)out.as<half_t>()[((size_t)b * Hq + h) * D + i];
                if (!(fabs(got - want) <= 2e-3 + 1e-3 * fabs(want))) wrong("another result: ");
            }
        }
}
int main() {
    signal(SIGSEGV, on_fault);
    signal(SIGBUS, on_fault);
    CASES
    return 0;
}
"""

# short, ragged and shared forms of every instantiation: lengths that end within a tile, at its end, at a page's end, in the last page of the cache
ATTENTION_CASES = {
    "fp16_narrow": """one<false, 64, 2, true>(64, 2, 3, 16, 0, 0, {1, 16, 17, 0, 33}); one<false, 64, 2, true>(64, 1, 20, 48, 0, 0, {49}); one<false, 64, 2, false>(16, 1, 2, 16, 0, 0, {5, 32});
                      one<false, 64, 2, false>(48, 2, 1, 32, 7, 0, {40}); one<false, 64, 2, true>(64, 1, 4, 16, 100, 3, {0, 300, 31, 0, 129, 1, 0});""",
    "fp16_128": """one<false, 128, 4, true>(128, 1, 4, 16, 0, 0, {31, 130}); one<false, 128, 4, false>(80, 2, 2, 16, 0, 0, {18}); one<false, 128, 4, false>(112, 1, 1, 64, 20, 2, {200, 65});
                   one<false, 128, 4, true>(128, 1, 17, 32, 0, 4, {260, 0, 64});""",
    "fp16_wide": """one<false, 256, 8, true>(256, 1, 2, 16, 0, 0, {33}); one<false, 256, 8, false>(144, 1, 16, 16, 0, 0, {16}); one<false, 256, 8, false>(240, 1, 1, 48, 0, 2, {150, 47});
                    one<false, 256, 8, true>(256, 1, 3, 32, 50, 2, {160, 0, 97});""",
    "q8_narrow": """one<true, 64, 1, false>(32, 2, 2, 16, 0, 0, {1, 33, 0}); one<true, 64, 2, true>(64, 1, 8, 16, 0, 0, {16, 129}); one<true, 64, 2, true>(64, 2, 1, 48, 33, 3, {250, 0, 0, 48, 96});""",
    "q8_128": """one<true, 128, 3, false>(96, 1, 2, 16, 0, 0, {31, 32}); one<true, 128, 4, true>(128, 1, 4, 64, 0, 0, {65}); one<true, 128, 4, true>(128, 1, 2, 16, 0, 3, {300, 1, 0, 128});
                 one<true, 128, 3, false>(96, 1, 1, 32, 40, 2, {200});""",
    "q8_wide": """one<true, 256, 5, false>(160, 1, 1, 16, 0, 0, {17}); one<true, 256, 6, false>(192, 1, 2, 16, 0, 0, {32}); one<true, 256, 7, false>(224, 1, 1, 48, 0, 2, {140});
                  one<true, 256, 8, true>(256, 1, 2, 16, 0, 2, {150, 0, 31}); one<true, 256, 8, true>(256, 1, 1, 32, 9, 0, {64});""",
}

CACHE = r"""
template <bool Q8> static void cache(uint32_t T, uint32_t Hq, uint32_t Hkv, uint32_t D, uint32_t n_rot, uint32_t ps, bool inter, bool prompt) {
    const uint32_t pages = (T + ps - 1) / ps + 1, qs = Hq * D + 8, ks = Hkv * D + 16;
    snprintf(what, sizeof what, "%s of %u tokens, %u + %u heads of %u, %u turned, pages of %u, %s, %s\n", prompt ? "prompt" : "rows", T, Hq, Hkv, D, n_rot, ps, inter ? "interleaved" : "halves", Q8 ? "Q8_0" : "fp16");
    const size_t values = (size_t)pages * Hkv * ps * D;
    // the last row ends with its last head
    Held q(2 * ((size_t)(T - 1) * qs + Hq * D)), to(2 * ((size_t)(T - 1) * qs + Hq * D)), k(2 * ((size_t)(T - 1) * ks + Hkv * D)), v(2 * ((size_t)(T - 1) * ks + Hkv * D)),
        kc(values * (Q8 ? 1 : 2)), vc(values * (Q8 ? 1 : 2)), kd(values / 16), vd(values / 16), pos(4 * T), slots(4 * T), freqs(4 * n_rot);
    fill(q.as<half_t>(), q.n / 2); fill(k.as<half_t>(), k.n / 2); fill(v.as<half_t>(), v.n / 2);
    for (uint32_t t = 0; t < T; ++t) {
        pos.as<int32_t>()[t] = (int32_t)rnd(100000);
        slots.as<int32_t>()[t] = t % 5 == 3 ? (t % 2 ? -1 : (int32_t)(pages * ps)) : (int32_t)(pages * ps - 1 - t);
    }
    for (uint32_t i = 0; i < n_rot / 2; ++i) freqs.as<double>()[i] = pow(10000.0, -2.0 * i / n_rot);
    RowsArgs a = {};
    a.q = q.as<half_t>(); a.k = k.as<half_t>(); a.v = v.as<half_t>(); a.q_stride = a.q_out_stride = qs; a.k_stride = a.v_stride = ks; a.q_out = to.as<half_t>();
    a.k_cache = kc.p; a.v_cache = vc.p; a.k_d = kd.as<half_t>(); a.v_d = vd.as<half_t>(); a.positions = pos.as<int32_t>(); a.slots = slots.as<int32_t>(); a.freqs = freqs.as<double>();
    a.Hq = Hq; a.Hkv = Hkv; a.chunks = D / 8; a.n_rot = n_rot; a.page_size = ps; a.n_slots = pages * ps; a.mscale = 1.0;
    a.heads_per_wg = kRowThreads / a.chunks;
    a.groups = (Hq + 2 * Hkv + a.heads_per_wg - 1) / a.heads_per_wg;
    const uint32_t items = (Hq + 2 * Hkv) * (a.chunks / 2), turns = (items + kRowThreads - 1) / kRowThreads, threads = ((items + turns - 1) / turns + 63) / 64 * 64;   // as launched
    if (prompt) run(threads, T, 1, 0, [&] { if (inter) prompt_kernel<true, Q8, true>(a); else prompt_kernel<true, Q8, false>(a); });
    else run(kRowThreads, a.groups * T, 1, 0, [&] { if (inter) rows_kernel<true, Q8, true>(a); else rows_kernel<true, Q8, false>(a); });
    for (uint32_t t = 0; t < T; ++t)
        for (uint32_t h = 0; h < Hq + 2 * Hkv; ++h)
            for (uint32_t i = 0; i < D; ++i) {
                const bool is_q = h < Hq, is_v = h >= Hq + Hkv;
                const uint32_t hk = is_q ? h : is_v ? h - Hq - Hkv : h - Hq;
                const half_t* row = (is_q ? a.q + t * (size_t)qs : is_v ? a.v + t * (size_t)ks : a.k + t * (size_t)ks) + hk * D;
                double want = (double)(float)row[i];
                if (!is_v && i < n_rot) {
                    const uint32_t p = inter ? i / 2 : i % (n_rot / 2);
                    const bool second = inter ? i & 1 : i >= n_rot / 2;
                    const double x0 = (double)(float)row[inter ? 2 * p : p], x1 = (double)(float)row[inter ? 2 * p + 1 : p + n_rot / 2], g = pos.as<int32_t>()[t] * freqs.as<double>()[p];
                    want = second ? x0 * sin(g) + x1 * cos(g) : x0 * cos(g) - x1 * sin(g);
                }
                double got, step = 2e-3 * fabs(want) + 1e-4;
                if (is_q) got = (double)(float)a.q_out[t * (size_t)qs + h * D + i];
                else {
                    const uint32_t slot = (uint32_t)slots.as<int32_t>()[t];
                    if (slot >= a.n_slots) continue;
                    const size_t r = ((size_t)(slot / ps) * Hkv + hk) * ps + slot % ps;
                    if (Q8) {
                        const float d = (float)(is_v ? a.v_d : a.k_d)[(r * D + i) / 32];
                        got = (double)(is_v ? vc : kc).as<int8_t>()[r * D + i] * d;
                        step += 0.6 * d;
                    } else got = (double)(float)(is_v ? vc : kc).as<half_t>()[r * D + i];
                }
                if (!(fabs(got - want) <= step)) wrong("another result: ");
            }
}
template <bool Q8> static void read(uint32_t Hkv, uint32_t D, uint32_t ps, std::vector<int32_t> lens, int32_t spare) {
    const uint32_t B = (uint32_t)lens.size();
    uint32_t most = 1, pages = 0, total = 0;
    for (int32_t n : lens) { most = std::max(most, (n + ps - 1) / ps); pages += (n + ps - 1) / ps; total += n; }
    snprintf(what, sizeof what, "reading back, %u sequences, %u rows, %u heads of %u, pages of %u, %s\n", B, total, Hkv, D, ps, Q8 ? "Q8_0" : "fp16");
    const size_t values = (size_t)pages * Hkv * ps * D;
    Held k(values * (Q8 ? 1 : 2)), v(values * (Q8 ? 1 : 2)), kd(values / 16), vd(values / 16), table(4 * (size_t)B * most), rows(4 * (B + 1)), ko((size_t)(total + spare) * Hkv * D * 2), vo((size_t)(total + spare) * Hkv * D * 2);
    for (size_t i = 0; i < k.n; ++i) { k.p[i] = (uint8_t)(rnd(64) + (Q8 ? 0 : i % 2 ? 0x20 : 0)); v.p[i] = k.p[i] ^ 1; }
    for (size_t i = 0; i < values / 32; ++i) kd.as<half_t>()[i] = vd.as<half_t>()[i] = (half_t)(0.25f * (1 + rnd(7)));
    memset(ko.p, 0xFF, ko.n); memset(vo.p, 0xFF, vo.n);
    int32_t at = 0, next = (int32_t)pages;
    for (uint32_t b = 0; b < B; ++b) {
        rows.as<int32_t>()[b] = at;
        at += lens[b];
        for (uint32_t i = 0; i < most; ++i) table.as<int32_t>()[b * most + i] = i < (lens[b] + ps - 1) / ps ? --next : -1;
    }
    rows.as<int32_t>()[B] = at;
    run(256, (total + spare) / 16 + B, (2 * Hkv * 16 * (D / 8) + 256 * kReadPieces - 1) / (256 * kReadPieces), 0, [&] {
        kv_read_kernel<Q8, false>(k.p, kd.as<half_t>(), v.p, vd.as<half_t>(), table.as<int32_t>(), most, rows.as<int32_t>(), ko.as<half_t>(), vo.as<half_t>(), total + spare, B, Hkv, D / 8, pages, ps);
    });
    for (uint32_t b = 0; b < B; ++b)
        for (int32_t t = 0; t < lens[b]; ++t)
            for (uint32_t i = 0; i < Hkv * D; ++i) {
                const size_t r = ((size_t)table.as<int32_t>()[b * most + t / ps] * Hkv + i / D) * ps + t % ps, from = r * D + i % D, dst = (size_t)(rows.as<int32_t>()[b] + t) * Hkv * D + i;
                const half_t want = Q8 ? (half_t)((float)k.as<int8_t>()[from] * (float)kd.as<half_t>()[from / 32]) : k.as<half_t>()[from];
                if (memcmp(&want, ko.as<half_t>() + dst, 2)) wrong("another key: ");
            }
    for (size_t i = (size_t)total * Hkv * D; i < ko.n / 2; ++i) if (ko.as<uint16_t>()[i] != 0xFFFF || vo.as<uint16_t>()[i] != 0xFFFF) wrong("rows behind the last sequence: ");
}
int main() {
    signal(SIGSEGV, on_fault);
    signal(SIGBUS, on_fault);
    for (int inter = 0; inter < 2; ++inter) {
        cache<false>(3, 5, 2, 64, 64, 16, inter, false); cache<false>(2, 40, 8, 128, 32, 16, inter, false); cache<false>(4, 1, 1, 16, 16, 48, inter, false);
        cache<false>(2, 3, 1, 80, 48, 16, inter, false); cache<false>(2, 1, 3, 256, 256, 16, inter, false);
        cache<true>(3, 7, 1, 96, 48, 16, inter, false); cache<true>(2, 2, 2, 32, 16, 32, inter, false); cache<true>(2, 16, 2, 256, 64, 16, inter, false); cache<true>(2, 33, 3, 64, 32, 16, inter, false);
        cache<false>(3, 5, 2, 64, 32, 16, inter, true); cache<false>(2, 3, 1, 80, 80, 16, inter, true); cache<false>(2, 1, 1, 16, 16, 16, inter, true); cache<false>(2, 40, 9, 128, 64, 16, inter, true);
        cache<true>(3, 5, 2, 64, 64, 16, inter, true); cache<true>(2, 17, 3, 128, 64, 48, inter, true); cache<true>(2, 3, 2, 256, 192, 16, inter, true);
    }
    read<false>(2, 64, 16, {1, 0, 17, 33}, 0); read<false>(1, 16, 48, {5, 48, 0, 0, 100}, 3); read<false>(3, 80, 16, {40}, 0); read<false>(1, 256, 32, {31, 32}, 1);
    read<true>(2, 64, 16, {0, 16, 1}, 0); read<true>(1, 96, 16, {33, 2}, 0); read<true>(2, 256, 64, {65, 0}, 2); read<true>(9, 32, 16, {3, 3, 3, 20}, 0);
    std::vector<int32_t> many;
    for (int i = 0; i < 150; ++i) many.push_back(i % 7 == 3 ? 0 : i % 5);
    read<false>(1, 16, 16, many, 0); read<true>(1, 32, 16, many, 5);
    return 0;
}
"""


def source(name, before):
    """The kernels of a source file (what stands in front of `before`, the host side), with the device header in place and what only the GPU's compiler takes replaced."""
    text = open(os.path.join(CSRC, name)).read()
    assert text.count(before) == 1
    text = text.split(before)[0].replace('#include "mxq_host.h"', "")
    header = open(os.path.join(CSRC, "mxq_device.h")).read().replace("#pragma once", "")
    asm = 'asm("v_cvt_f16_f32 %0, %1" : "=v"(r) : "v"(v));'
    assert header.count(asm) == 1
    header = header.replace(asm, "const _Float16 shim_h = (_Float16)v; uint16_t shim_u; memcpy(&shim_u, &shim_h, 2); r = shim_u;")
    text = text.replace('#include "mxq_device.h"', header)
    for name in ("lds", "sums"):
        text = text.replace("extern __shared__ float %s[];" % name, "float* const %s = reinterpret_cast<float*>(shim_lds);" % name)
    assert "extern __shared__" not in text
    return text.replace("__attribute__((address_space(4)))", "") + "}  // namespace mxq\n"


def build_and_run(tmp_path, program):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(program)
    subprocess.run([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), "-x", "c++", "-D__HIP_PLATFORM_AMD__", "-std=c++17", "-O1", "-w", "-I", "/opt/rocm/include", str(src), "-o", str(exe)], check=True)
    p = subprocess.run([str(exe)], capture_output=True, text=True)
    assert p.returncode == 0, (p.returncode, p.stdout + p.stderr)


def test_rows_and_cache(tmp_path):
    build_and_run(tmp_path, SHIM + source("kv_cache.hip", "// ---------------------------------------------------------------- argument checks").replace(
        "constexpr uint32_t kPromptTokens", "#if 0\nconstexpr uint32_t kPromptTokens").replace("// Reading back: a workgroup", "#endif\n// Reading back: a workgroup") + CHECK + CACHE)


@pytest.mark.parametrize("form", sorted(ATTENTION_CASES))
def test_attention(tmp_path, form):
    build_and_run(tmp_path, SHIM + source("attn_decode.hip", "// Short sequences take a workgroup each.") + CHECK + ATTENTION.replace("CASES", ATTENTION_CASES[form]))
