// routing.hip — MoE routing and packing on the device, so that a layer never waits for the host
// between the router and the expert kernels:
//   router logits + softmax + top-k + renormalise + ascending-id order   src/ops/moe.cpp:22-216
//   softmax + top-k from logits already on the device                     src/ops/moe.cpp:366-412
//   packing arrays for one token                                          src/ops/moe.cpp:423-446
//   packing arrays for T tokens: stable counting sort by expert           src/model/qwen3moe_pack.cpp:5-31
//   softmax or sigmoid scores, a bias, groups, top-k from logits          (no counterpart)
#include "mxq_device.h"
#include "mxq_host.h"

namespace mxq {

// ---------------------------------------------------------------- router logits
// logit[t, e] = sum_h W_gate[e, h] * x[t, h], fp32 weights and sums.  One summation order for every call, whatever its batch,
// sizes and alignments, so that a token is routed alike alone, in a decode batch and in a prompt:
//   lane l takes the elements 4 l .. 4 l + 3 of every 256-element piece, router_dot4 over the four, pieces added in order;
//   the 64 lane sums meet in a balanced tree of neighbours.
// (32 products a lane at hidden 2048, then six levels: rms error against 64-bit sums 9.6e-8, maximum 5.4e-7, logits of unit variance.
// One fp32 MFMA accumulator per output, a chain of 128 or 256 products, takes 17 us where this takes 25 to 27 (2048 tokens, 128
// experts) but has rms 2.2e-7 to 2.9e-7 and maximum 1.8e-6: near ties are routed otherwise.)
__device__ __forceinline__ float router_dot4(const float4& w, const float (&x)[4]) {
    return __builtin_fmaf(w.w, x[3], __builtin_fmaf(w.z, x[2], __builtin_fmaf(w.x, x[0], w.y * x[1])));
}

// Halves N values per lane: the lane keeps the odd or the even ones (sel) and adds its partner's, or, with one value left, adds
// the partner's.  Level d pairs neighbouring groups of 2^d lanes.  DPP has no exchange at distance 4 or 8, but mirrors of 8 and 16
// lanes; `sel` of the lower levels is chosen so that mirrored lanes hold the same values.
template <int N, int D>
__device__ __forceinline__ void router_level(float (&v)[N], float (&o)[N > 1 ? N / 2 : 1], uint32_t lane) {
    auto partner = [](float x) {
        if constexpr (D == 0) return dpp_f<0xB1>(x);
        else if constexpr (D == 1) return dpp_f<0x4E>(x);
        else if constexpr (D == 2) return dpp_f<0x141>(x);
        else if constexpr (D == 3) return dpp_f<0x140>(x);
        else return __shfl_xor(x, 1 << D);
    };
    if constexpr (N == 1) {
        o[0] = v[0] + partner(v[0]);
    } else {
        const bool sel = ((D == 0 ? lane ^ (lane >> 2) : D == 1 ? (lane >> 1) ^ (lane >> 2) : D == 2 ? (lane >> 2) ^ (lane >> 3) : lane >> D) & 1u) != 0u;
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const float keep = sel ? v[2 * i + 1] : v[2 * i], send = sel ? v[2 * i] : v[2 * i + 1];
            o[i] = keep + partner(send);
        }
    }
}
template <int N, int D = 0>
__device__ __forceinline__ float router_tree(float (&v)[N], uint32_t lane) {
    float o[N > 1 ? N / 2 : 1];
    router_level<N, D>(v, o, lane);
    if constexpr (D == 5) return o[0];
    else return router_tree<(N > 1 ? N / 2 : 1), D + 1>(o, lane);
}

// One wave = MT tokens x NE experts, MT NE accumulators per lane (a power of two up to 64).  U: pieces whose loads are requested
// together.  The waves of a workgroup take neighbouring token tiles of the same experts.  Bound by: the load latency of a row at a
// few tokens, five vector instructions per four products at many (2048 tokens, 128 experts, hidden 2048: 17 us of issue, 25 to
// 27 measured; one wave per output, which reads W once per token: 140).
template <int MT, int NE, int U>
__global__ __launch_bounds__(256) void router_logits_kernel(const half_t* __restrict__ x, const float* __restrict__ W, float* __restrict__ logits, uint32_t T,
                                                            uint32_t hidden, uint32_t E) {
    constexpr int P = MT * NE;
    static_assert((P & (P - 1)) == 0 && P <= 64, "one result per lane at most");
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t tile = blockIdx.x * (blockDim.x / 64u) + (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t t_tiles = (T + MT - 1u) / MT, e0 = tile / t_tiles * NE, t0 = tile % t_tiles * MT;
    if (e0 >= E) return;
    const uint2* xr[MT];
    const float4* wr[NE];
#pragma unroll
    for (int m = 0; m < MT; ++m) xr[m] = reinterpret_cast<const uint2*>(x + (size_t)(t0 + m < T ? t0 + m : T - 1u) * hidden);   // uniform; piece c: xr[64 c + lane]
#pragma unroll
    for (int n = 0; n < NE; ++n) wr[n] = reinterpret_cast<const float4*>(W + (size_t)(e0 + n < E ? e0 + n : E - 1u) * hidden);
    float acc[P];
#pragma unroll
    for (int p = 0; p < P; ++p) acc[p] = 0.f;
    struct Piece {
        uint2 x[MT];
        float4 w[NE];
    };
    auto load = [&](uint32_t c, Piece& p) {
#pragma unroll
        for (int n = 0; n < NE; ++n) p.w[n] = wr[n][64u * c + lane];
#pragma unroll
        for (int m = 0; m < MT; ++m) p.x[m] = xr[m][64u * c + lane];
    };
    auto add = [&](const Piece& p) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const float v[4] = {h2f(p.x[m].x & 0xFFFFu), h2f(p.x[m].x >> 16), h2f(p.x[m].y & 0xFFFFu), h2f(p.x[m].y >> 16)};
#pragma unroll
            for (int n = 0; n < NE; ++n) acc[m * NE + n] += router_dot4(p.w[n], v);
        }
    };
    const uint32_t n_full = hidden / 256u;
    const bool last = n_full * 256u + lane * 4u < hidden;   // the lanes that take part in the last, partial piece
    Piece end{};
    if (P <= 4 && last) load(n_full, end);                  // few outputs: requested ahead of everything else
    for (uint32_t c = 0; c < n_full; c += U) {
        Piece p[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (U == 1 || c + u < n_full) load(c + u, p[u]);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (U == 1 || c + u < n_full) add(p[u]);
    }
    if (last) {
        if (P > 4) load(n_full, end);
        add(end);
    }
    const float sum = router_tree(acc, lane);
    // which value this lane has kept: one bit per halving level, the level's `sel`
    const uint32_t key = ((lane ^ (lane >> 2)) & 1u) | (((lane >> 1) ^ (lane >> 2)) & 1u) << 1 | (((lane >> 2) ^ (lane >> 3)) & 1u) << 2 | (lane & 56u);
    const uint32_t k = key & (P - 1u), t = t0 + k / NE, e = e0 + k % NE;
    if (lane < P && t < T && e < E) logits[(size_t)t * E + e] = sum;
}

template <int MT, int NE, int U, uint32_t WV>
static int launch_router(hipStream_t st, const half_t* x, const float* W, float* logits, uint32_t T, uint32_t hidden, uint32_t E) {
    const uint32_t tiles = ((T + MT - 1u) / MT) * ((E + NE - 1u) / NE);
    hipLaunchKernelGGL((router_logits_kernel<MT, NE, U>), dim3((tiles + WV - 1u) / WV), dim3(64u * WV), 0, st, x, W, logits, T, hidden, E);
    return launch_status();
}
// The tile by the number of outputs: small tiles spread few outputs over the CUs, large ones read the rows less often.  Times with
// the top-k behind it, us, 1 x 1 (one wave per workgroup) / 2 x 2 / 4 x 4 / 8 x 8: 128 experts, hidden 2048: 16 tokens 6.8 / 6.9 / 7.9 /
// 13, 64 tokens 9.7 / 8.0 / 8.1 / 13, 333 tokens 26 / 16 / 11.9 / 13, 1024 tokens 67 / 35 / 21.5 / 18; 32 experts, hidden 2880:
// one token 4.8 / 6.2 / 7.5 / 14, 512 tokens 17 / 11 / 8.7 / 15, 2048 tokens 54 / 29 / 16.9 / 15.6.
static int launch_router_logits(hipStream_t st, const half_t* x, const float* W, float* logits, uint32_t T, uint32_t hidden, uint32_t E) {
    const uint32_t n = T * E;   // at most 65535 x 1024
    if (n <= 2048u) return launch_router<1, 1, 8, 1>(st, x, W, logits, T, hidden, E);
    if (n <= 8192u) return launch_router<2, 2, 4, 4>(st, x, W, logits, T, hidden, E);
    if (n < 65536u) return launch_router<4, 4, 1, 4>(st, x, W, logits, T, hidden, E);
    return launch_router<8, 8, 1, 4>(st, x, W, logits, T, hidden, E);
}

// ---------------------------------------------------------------- softmax + top-k
constexpr int kMaxTopK = 64;

__device__ __forceinline__ float wave_max_f(float v) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}
// maximum over the wave in a scalar register: DPP inside the rows, row broadcasts across them, lane 63 holds the result
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    auto step = [&](uint32_t o) { v = o > v ? o : v; };
    step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));
    step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));
    step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, true));
    step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, true));
    step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false));
    step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false));
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// One wave per token, lane l holds the experts l, l + 64, .. (NJ of them).  p = softmax(logits); K rounds of a wave-wide
// maximum over the float bits of p (monotonic for p >= 0; 1 is added so that 0 can mark an expert that is taken), the
// highest id among exact ties; then every winner renormalises its own weight and finds its place by counting the winners
// with a lower id.  No barrier, no LDS: 2048 tokens of 128 experts, k = 8, take 3.8 us where one workgroup per token with
// two barriers per round and a serial sort took 11.8; one token of 32 experts 2.3 (4.4).
template <class LogitT, int NJ>
__global__ __launch_bounds__(256) void topk_kernel(const LogitT* logits, int32_t* topk_idx, half_t* topk_w, uint32_t E, uint32_t K, uint32_t n_tokens) {
    const uint32_t lane = threadIdx.x & 63u, t = blockIdx.x * 4u + (threadIdx.x >> 6);
    if (t >= n_tokens) return;
    const LogitT* lg = logits + (size_t)t * E;
    float p[NJ];
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        const uint32_t e = lane + 64u * j;
        p[j] = e < E ? load_act(lg + e) : -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) m = fmaxf(m, p[j]);
    m = wave_max_f(m);
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        p[j] = lane + 64u * j < E ? __expf(p[j] - m) : 0.f;
        s += u2f((uint32_t)__builtin_amdgcn_readlane((int)f2u(group_sum<64>(p[j])), 63));
    }
    uint32_t key[NJ];
    unsigned long long taken[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        p[j] = p[j] / s;
        const uint32_t bits = f2u(p[j]) < 0xFFFFFFFEu ? f2u(p[j]) : 0xFFFFFFFEu;   // a NaN of all ones stays a key: every round has a winner
        key[j] = lane + 64u * j < E ? bits + 1u : 0u;
        taken[j] = 0ull;
    }
    float ren = 0.f;
    for (uint32_t kk = 0; kk < K; ++kk) {
        uint32_t best = key[0];
#pragma unroll
        for (int j = 1; j < NJ; ++j) best = key[j] > best ? key[j] : best;
        const uint32_t win = wave_max_u32(best);
        ren += u2f(win - 1u);
        bool open = true;
#pragma unroll
        for (int j = NJ - 1; j >= 0; --j) {
            const unsigned long long hit = open ? __ballot(key[j] == win && key[j] != 0u) : 0ull;
            if (hit) {
                const uint32_t l = 63u - (uint32_t)__builtin_clzll(hit);
                taken[j] |= 1ull << l;
                if (lane == l) key[j] = 0u;
                open = false;
            }
        }
    }
    const float inv = 1.0f / ren;
    uint32_t below = 0;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        if ((taken[j] >> lane) & 1ull) {
            const uint32_t at = below + (uint32_t)__builtin_popcountll(taken[j] & ((1ull << lane) - 1ull));
            topk_idx[(size_t)t * K + at] = (int32_t)(lane + 64u * j);
            float w = p[j] * inv;
            asm volatile("" : "+v"(w));   // an fp32 value first: the compiler would round the product to fp16 at once
            topk_w[(size_t)t * K + at] = (half_t)w;
        }
        below += (uint32_t)__builtin_popcountll(taken[j]);
    }
}

template <class LogitT>
static int launch_topk(hipStream_t st, const LogitT* logits, int32_t* topk_idx, half_t* topk_w, uint32_t E, uint32_t K, uint32_t n_tokens) {
    const dim3 grid((n_tokens + 3) / 4), block(256);
    if (E <= 64) hipLaunchKernelGGL((topk_kernel<LogitT, 1>), grid, block, 0, st, logits, topk_idx, topk_w, E, K, n_tokens);
    else if (E <= 128) hipLaunchKernelGGL((topk_kernel<LogitT, 2>), grid, block, 0, st, logits, topk_idx, topk_w, E, K, n_tokens);
    else if (E <= 256) hipLaunchKernelGGL((topk_kernel<LogitT, 4>), grid, block, 0, st, logits, topk_idx, topk_w, E, K, n_tokens);
    else hipLaunchKernelGGL((topk_kernel<LogitT, 16>), grid, block, 0, st, logits, topk_idx, topk_w, E, K, n_tokens);
    return launch_status();
}

// ---------------------------------------------------------------- scores, bias, groups, top-k
// A 64-bit number as an unsigned one of the same order; every NaN is 2^32, below all numbers, and an upper half of 0 is left for experts that are out.
__device__ __forceinline__ uint64_t order_of(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return v == v ? (b >> 63 ? ~b : b | 1ull << 63) : 1ull << 32;
}
__device__ __forceinline__ double number_of(uint64_t k) {
    return k == 1ull << 32 ? __builtin_nan("") : __builtin_bit_cast(double, k >> 63 ? k & ~(1ull << 63) : ~k);
}
template <int CTRL, int ROW_MASK = 0xF, bool BOUND = true>
__device__ __forceinline__ uint64_t dpp_u64(uint64_t v) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROW_MASK, 0xF, BOUND), hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROW_MASK, 0xF, BOUND);
    return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t lane_u64(uint64_t v, int lane) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}
__device__ __forceinline__ double wave_sum_f64(double v) {
    auto step = [&](uint64_t o) { v += __builtin_bit_cast(double, o); };
    step(dpp_u64<0xB1>(__builtin_bit_cast(uint64_t, v)));
    step(dpp_u64<0x4E>(__builtin_bit_cast(uint64_t, v)));
    step(dpp_u64<0x141>(__builtin_bit_cast(uint64_t, v)));
    step(dpp_u64<0x140>(__builtin_bit_cast(uint64_t, v)));
    step(dpp_u64<0x142, 0xA, false>(__builtin_bit_cast(uint64_t, v)));
    step(dpp_u64<0x143, 0xC, false>(__builtin_bit_cast(uint64_t, v)));
    return __builtin_bit_cast(double, lane_u64(__builtin_bit_cast(uint64_t, v), 63));
}
__device__ __forceinline__ float wave_max_dpp(float v) {
    v = fmaxf(v, dpp_f<0xB1>(v));
    v = fmaxf(v, dpp_f<0x4E>(v));
    v = fmaxf(v, dpp_f<0x141>(v));
    v = fmaxf(v, dpp_f<0x140>(v));
    v = fmaxf(v, u2f((uint32_t)__builtin_amdgcn_update_dpp((int)f2u(-INFINITY), (int)f2u(v), 0x142, 0xA, 0xF, false)));
    v = fmaxf(v, u2f((uint32_t)__builtin_amdgcn_update_dpp((int)f2u(-INFINITY), (int)f2u(v), 0x143, 0xC, 0xF, false)));
    return u2f((uint32_t)__builtin_amdgcn_readlane((int)f2u(v), 63));
}

struct RouteArgs {
    const void* logits;
    const float* bias;
    int32_t* topk_idx;
    half_t* topk_w;
    uint32_t n_tokens, E, K, n_groups, size, size_inv, kept, lanes, flags;   // size: experts of a group, size_inv = ceil(2^32 / size); lanes: of a wave for each group
    float scale;
    bool wide;               // a lane's logits are loaded at once
};

// The two largest of two pairs (first >= second).
__device__ __forceinline__ void merge_two(uint64_t& first, uint64_t& second, uint64_t f, uint64_t s) {
    const uint64_t low = f < first ? f : first, more = s > second ? s : second;
    first = f > first ? f : first;
    second = low > more ? low : more;
}

// One wave a token, lane l holds experts NJ l .. NJ l + NJ - 1: scores in 64 bits and, as integers of the same order, what they are chosen by.  K rounds of a maximum over the wave: the upper halves of the
// keys decide, and where several have the largest the lower halves and then the lowest id; who is taken is kept in scalar masks, which are the conditions of what follows.  The chosen meet in LDS and lane i
// writes the i-th.  4096 tokens to 8 of 256 experts in groups 8.8 us (rounds over whole keys 11.5, shifted masks 10.5, every lane writing its own 10.2, bias by bias 9.4), one token of 128 experts 2.9 (3.5, 3.2, 3.0).
// Bound by the vector instructions and, for few tokens, by their latency one after the other.
template <int NJ>
__global__ __launch_bounds__(256) void route_kernel(RouteArgs a) {
    __shared__ uint64_t choice[4][NJ * 64];
    __shared__ uint32_t ids[4][64];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, t = blockIdx.x * 4u + wave, e0 = lane * NJ;
    if (t >= a.n_tokens) return;          // no barriers: a wave's LDS is its own
    float x[NJ];
    const size_t row = (size_t)t * a.E + e0;
    typedef float floats __attribute__((ext_vector_type(NJ)));
    typedef _Float16 halves __attribute__((ext_vector_type(NJ)));
#pragma unroll
    for (int j = 0; j < NJ; ++j) x[j] = -INFINITY;
    if (a.wide) {            // E is a multiple of NJ
        if (e0 < a.E) {
            if (a.flags & MX_ROUTE_F32) {
                const floats v = *reinterpret_cast<const floats*>(static_cast<const float*>(a.logits) + row);
#pragma unroll
                for (int j = 0; j < NJ; ++j) x[j] = v[j];
            } else {
                const halves v = *reinterpret_cast<const halves*>(static_cast<const half_t*>(a.logits) + row);
#pragma unroll
                for (int j = 0; j < NJ; ++j) x[j] = (float)v[j];
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < NJ; ++j)
            if (e0 + j < a.E) x[j] = a.flags & MX_ROUTE_F32 ? static_cast<const float*>(a.logits)[row + j] : (float)static_cast<const half_t*>(a.logits)[row + j];
    }
    float add[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) add[j] = 0.f;
    if (a.wide && a.bias) {
        typedef float floats_anywhere __attribute__((ext_vector_type(NJ), aligned(4)));
        if (e0 < a.E) {
            const floats_anywhere v = *reinterpret_cast<const floats_anywhere*>(a.bias + e0);
#pragma unroll
            for (int j = 0; j < NJ; ++j) add[j] = v[j];
        }
    } else if (a.bias) {
#pragma unroll
        for (int j = 0; j < NJ; ++j)
            if (e0 + j < a.E) add[j] = a.bias[e0 + j];
    }
    double score[NJ];
    if (a.flags & MX_ROUTE_SIGMOID) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) score[j] = 1.0 / (1.0 + exp(-(double)x[j]));
    } else {
        float m = x[0];
#pragma unroll
        for (int j = 1; j < NJ; ++j) m = fmaxf(m, x[j]);
        m = wave_max_dpp(m);
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            score[j] = x[j] == -INFINITY ? 0.0 : exp((double)x[j] - (double)m);
            sum += score[j];
        }
        sum = wave_sum_f64(sum);
        const double inv = sum == 0.0 ? 0.0 : 1.0 / sum;
#pragma unroll
        for (int j = 0; j < NJ; ++j) score[j] *= inv;
    }
    uint64_t key[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) key[j] = e0 + j < a.E ? order_of(a.bias ? score[j] + (double)add[j] : score[j]) : 0ull;
    if (a.n_groups > 1) {
        uint64_t first = 0, second = 0;
        const bool whole = a.size % NJ == 0 && (a.size / NJ & (a.size / NJ - 1)) == 0;    // groups of whole lanes, a power of two of them
        if (whole) {
            const uint32_t of = a.size / NJ;
#pragma unroll
            for (int j = 0; j < NJ; ++j) merge_two(first, second, key[j], 0ull);
            // equal within 2, 4, 8 lanes, a mirror brings the other half of twice as many
            if (of > 1) merge_two(first, second, dpp_u64<0xB1>(first), dpp_u64<0xB1>(second));
            if (of > 2) merge_two(first, second, dpp_u64<0x4E>(first), dpp_u64<0x4E>(second));
            if (of > 4) merge_two(first, second, dpp_u64<0x141>(first), dpp_u64<0x141>(second));
            if (of > 8) merge_two(first, second, dpp_u64<0x140>(first), dpp_u64<0x140>(second));
            if (of > 16) merge_two(first, second, __shfl_xor(first, 16), __shfl_xor(second, 16));
        } else {
            // by `lanes` lanes each, from LDS
#pragma unroll
            for (int j = 0; j < NJ; ++j) choice[wave][e0 + j] = key[j];
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            const uint32_t group = lane / a.lanes;
            if (group < a.n_groups)
                for (uint32_t i = lane - group * a.lanes; i < a.size; i += a.lanes) merge_two(first, second, choice[wave][group * a.size + i], 0ull);
            for (uint32_t d = 1; d < a.lanes; d <<= 1) merge_two(first, second, __shfl_xor(first, d), __shfl_xor(second, d));
        }
        const uint32_t of = whole ? a.size / NJ : a.lanes, own = lane / of;               // lanes of a group
        const uint64_t worth = a.flags & MX_ROUTE_TOP2 && a.size > 1 ? order_of(number_of(first) + number_of(second)) : first;
        uint32_t better = 0;
        for (uint32_t g = 0; g < a.n_groups; ++g) {
            const uint64_t other = lane_u64(worth, (int)(g * of));
            better += other > worth || (other == worth && g < own) ? 1u : 0u;
        }
        const bool in = own < a.n_groups && better < a.kept;
        if (whole) {
#pragma unroll
            for (int j = 0; j < NJ; ++j) key[j] = in ? key[j] : 0ull;
        } else {
            const uint64_t kept = __ballot(in && lane % of == 0);                          // bit g * of
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const uint32_t g = a.size == 1u ? e0 + j : __umulhi(e0 + j, a.size_inv);
                if (!(kept >> (g * of & 63u) & 1ull)) key[j] = 0ull;
            }
        }
    }
    uint32_t high[NJ];
    uint64_t taken[NJ];      // bit l: lane l's
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        high[j] = (uint32_t)(key[j] >> 32);
        taken[j] = 0ull;
    }
    for (uint32_t kk = 0; kk < a.K; ++kk) {
        uint32_t best = high[0];
#pragma unroll
        for (int j = 1; j < NJ; ++j) best = max(best, high[j]);
        const uint32_t top = wave_max_u32(best);
        uint64_t hit[NJ];
        uint32_t n = 0;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            hit[j] = __ballot(high[j] == top);
            n += (uint32_t)__builtin_popcountll(hit[j]);
        }
        if (n != 1) {
            uint32_t low = 0;
#pragma unroll
            for (int j = 0; j < NJ; ++j) low = max(low, high[j] == top ? (uint32_t)key[j] : 0u);
            low = wave_max_u32(low);
            uint64_t any = 0;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                hit[j] = __ballot(high[j] == top && (uint32_t)key[j] == low);
                any |= hit[j];
            }
            uint64_t lane_bit = any & (0ull - any);                   // the lowest lane, and of its experts the first
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                hit[j] &= lane_bit;
                lane_bit &= ~hit[j];
            }
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            taken[j] |= hit[j];
            high[j] = __builtin_amdgcn_inverse_ballot_w64(hit[j]) ? 0u : high[j];
        }
    }
    double factor = (double)a.scale;
    if (a.flags & MX_ROUTE_RENORM) {
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < NJ; ++j) sum += __builtin_amdgcn_inverse_ballot_w64(taken[j]) ? score[j] : 0.0;
        factor /= wave_sum_f64(sum) + 1e-20;
    }
    uint32_t at = 0;         // chosen experts of lower lanes
#pragma unroll
    for (int j = 0; j < NJ; ++j) at = (uint32_t)__builtin_amdgcn_mbcnt_hi((uint32_t)(taken[j] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)taken[j], at));
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");                                   // the groups' keys have been read
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < NJ; ++j)
        if (__builtin_amdgcn_inverse_ballot_w64(taken[j])) {
            choice[wave][at] = __builtin_bit_cast(uint64_t, score[j]);
            ids[wave][at++] = e0 + j;
        }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    if (lane < a.K) {
        a.topk_idx[(size_t)t * a.K + lane] = (int32_t)ids[wave][lane];
        a.topk_w[(size_t)t * a.K + lane] = (half_t)(__builtin_bit_cast(double, choice[wave][lane]) * factor);
    }
}

// ---------------------------------------------------------------- packing
// One token (src/ops/moe.cpp:423-446): offsets by counting, identity order.
__global__ void pack_decode_kernel(const int32_t* topk_idx, const half_t* topk_w, uint32_t* expert_offsets, int32_t* sorted_idx, int32_t* tk_to_packed,
                                   half_t* weights_packed, uint32_t E, uint32_t K) {
    // thread e counts the slots routed below e
    for (uint32_t e = threadIdx.x; e <= E; e += blockDim.x) {
        uint32_t below = 0;
        for (uint32_t kk = 0; kk < K; ++kk) below += ((uint32_t)topk_idx[kk] < e) ? 1u : 0u;
        expert_offsets[e] = below;
    }
    for (uint32_t kk = threadIdx.x; kk < K; kk += blockDim.x) {
        sorted_idx[kk] = 0;
        tk_to_packed[kk] = (int32_t)kk;
        weights_packed[kk] = topk_w[kk];
    }
}

// T tokens: stable counting sort of the T*K slots by expert id, in one launch.  Workgroup g sorts the slots of the Q experts
// from e0 = Q g on: it reads all ids, its waves a contiguous range each, counts the slots of every one of its experts (a
// ballot each) and those of all experts below e0, which is where its own begin; the counts of the waves meet in LDS, and in a
// second round over its ids a lane whose slot is one of the workgroup's knows its place.  So nothing passes between workgroups, at the
// price of reading the ids E / Q times, from L2.  With at most R = 4 or 16 slots a lane the ids stay in registers
// between the rounds (R = 0: read again).  One expert a workgroup up to 128 experts (128 experts, 16384 slots 10.5 us on cold caches,
// four experts a workgroup 14.6), four beyond, where the ids would be read too often.  Bound by the vector instructions per 64 slots.  us, one
// workgroup that ranks the slots of all experts with a ballot per id bit (bound by the pipes of its one CU) / this: 32 experts, 128
// slots 4.7 / 4.0; 128 experts, 2664 slots 6.9 / 4.7, 16384 slots 17.4 / 7.4, 65536 slots 101 / 21; 256 experts, 16384 slots 18.7 / 10.9;
// 1024 experts, 256 slots 10.2 / 3.7, 36000 slots 72 / 16.
template <int R, uint32_t Q>
__global__ __launch_bounds__(1024) void pack_kernel(const int32_t* __restrict__ topk_idx, const uint16_t* __restrict__ topk_w, uint32_t n, uint32_t K, uint32_t E,
                                                    uint32_t* __restrict__ expert_offsets, int32_t* __restrict__ sorted_idx,
                                                    uint16_t* __restrict__ weights_packed, int32_t* __restrict__ tk_to_packed) {
    __shared__ uint32_t counts[16][Q + 1];   // [wave]: slots of the Q experts, slots of experts below
    const uint32_t tid = threadIdx.x, lane = tid & 63u, n_waves = blockDim.x / 64u;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
    const uint32_t e0 = blockIdx.x * Q, n_own = E - e0 < Q ? E - e0 : Q;
    const uint32_t batches = (n + 63u) / 64u, per = (batches + n_waves - 1u) / n_waves;   // of 64 slots; a wave's
    const uint64_t lo64 = (uint64_t)wave * per * 64u, hi64 = lo64 + (uint64_t)per * 64u;
    const uint32_t lo = lo64 < n ? (uint32_t)lo64 : n, hi = hi64 < n ? (uint32_t)hi64 : n;
    constexpr int U = R ? R : 4;
    uint32_t id[U];
    auto load = [&](uint32_t c) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t i = c + 64u * u + lane;
            id[u] = i < hi ? (uint32_t)topk_idx[i] : 0xFFFFFFFFu;   // no expert's: slots without an expert of the bank are left out
        }
    };
    uint32_t cnt[Q] = {}, below = 0;
    auto count = [&]() {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            below += (uint32_t)__popcll(__ballot(id[u] < e0));
#pragma unroll
            for (uint32_t q = 0; q < Q; ++q) cnt[q] += (uint32_t)__popcll(__ballot(id[u] == e0 + q));
        }
    };
    if constexpr (R > 0) {
        load(lo);
        count();
    } else {
        for (uint32_t c = lo; c < hi; c += 64u * U) {
            load(c);
            count();
        }
    }
    if (lane <= Q) {
        uint32_t v = below;
#pragma unroll
        for (uint32_t q = 0; q < Q; ++q) v = lane == q ? cnt[q] : v;
        counts[wave][lane] = v;
    }
    __syncthreads();
    // lane q <= Q: the sum over all waves and the one over the waves before this one
    uint32_t all = 0, before = 0;
    for (uint32_t w = 0; w < n_waves; ++w) {
        const uint32_t v = lane <= Q ? counts[w][lane] : 0u;
        all += v;
        before += w < wave ? v : 0u;
    }
    uint32_t at[Q], first = (uint32_t)__builtin_amdgcn_readlane((int)all, (int)Q);
#pragma unroll
    for (uint32_t q = 0; q < Q; ++q) {
        if (tid == 0 && q < n_own) expert_offsets[e0 + q] = first;
        at[q] = first + (uint32_t)__builtin_amdgcn_readlane((int)before, (int)q);
        if (q < n_own) first += (uint32_t)__builtin_amdgcn_readlane((int)all, (int)q);
    }
    if (tid == 0 && e0 + n_own == E) expert_offsets[E] = first;
    const bool small = n <= 65536u;
    const uint32_t inv = K > 1u ? 0xFFFFFFFFu / K + 1u : 0u;   // slot / K by a multiplication: exact below 2^16
    auto place = [&](uint32_t c) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t i = c + 64u * u + lane, rel = id[u] - e0;
            if (__ballot(rel < n_own) == 0ull) continue;
            uint32_t p = 0;
#pragma unroll
            for (uint32_t q = 0; q < Q; ++q) {
                const unsigned long long m = __ballot(rel == q);
                const uint32_t r = at[q] + (uint32_t)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u));
                p = rel == q ? r : p;
                at[q] += (uint32_t)__popcll(m);
            }
            if (rel < n_own) {
                sorted_idx[p] = (int32_t)(K == 1u ? i : small ? __umulhi(i, inv) : i / K);
                weights_packed[p] = topk_w[i];
                tk_to_packed[i] = (int32_t)p;
            }
        }
    };
    if constexpr (R > 0) {
        place(lo);
    } else {
        for (uint32_t c = lo; c < hi; c += 64u * U) {
            load(c);
            place(c);
        }
    }
}

}  // namespace mxq

using namespace mxq;

extern "C" {

int mx_moe_topk_from_logits(mx_stream_t s, const uint16_t* logits, int32_t* topk_idx, uint16_t* topk_w, uint32_t E, uint32_t K, uint32_t n_tokens) {
    MX_REQUIRE_PTR(logits); MX_REQUIRE_PTR(topk_idx); MX_REQUIRE_PTR(topk_w);
    MX_REQUIRE_SHAPE(E > 0 && E <= 1024 && K > 0 && K <= E && K <= (uint32_t)kMaxTopK && n_tokens > 0);
    return launch_topk(as_stream(s), reinterpret_cast<const half_t*>(logits), topk_idx, reinterpret_cast<half_t*>(topk_w), E, K, n_tokens);
}

int mx_moe_router(mx_stream_t s, const uint16_t* x, const float* W_gate, int32_t* topk_idx, uint16_t* topk_w, uint32_t n_tokens, uint32_t hidden,
                  uint32_t n_experts, uint32_t k, float* logits_ws) {
    MX_REQUIRE_PTR(x); MX_REQUIRE_PTR(W_gate); MX_REQUIRE_PTR(topk_idx); MX_REQUIRE_PTR(topk_w); MX_REQUIRE_PTR(logits_ws);
    MX_REQUIRE_SHAPE(n_tokens > 0 && n_tokens <= 65535 && hidden > 0 && hidden % 4 == 0 && n_experts > 0 && n_experts <= 1024 && k > 0 && k <= n_experts &&
                     k <= (uint32_t)kMaxTopK);
    MX_REQUIRE_ALIGN(x, 8); MX_REQUIRE_ALIGN(W_gate, 16);
    hipStream_t st = as_stream(s);
    if (int rc = launch_router_logits(st, reinterpret_cast<const half_t*>(x), W_gate, logits_ws, n_tokens, hidden, n_experts)) return rc;
    return launch_topk(st, (const float*)logits_ws, topk_idx, reinterpret_cast<half_t*>(topk_w), n_experts, k, n_tokens);
}

int mx_moe_router_logits(mx_stream_t s, const uint16_t* x, const float* W_gate, float* logits, uint32_t n_tokens, uint32_t hidden, uint32_t n_experts) {
    MX_REQUIRE_PTR(x); MX_REQUIRE_PTR(W_gate); MX_REQUIRE_PTR(logits);
    MX_REQUIRE_SHAPE(n_tokens > 0 && n_tokens <= 65535 && hidden > 0 && hidden % 4 == 0 && n_experts > 0 && n_experts <= 1024);
    MX_REQUIRE_ALIGN(x, 8); MX_REQUIRE_ALIGN(W_gate, 16); MX_REQUIRE_ALIGN(logits, 4);
    return launch_router_logits(as_stream(s), reinterpret_cast<const half_t*>(x), W_gate, logits, n_tokens, hidden, n_experts);
}

int mx_moe_route(mx_stream_t s, const void* logits, const float* bias, int32_t* topk_idx, uint16_t* topk_w, uint32_t n_tokens, uint32_t n_experts, uint32_t k,
                 uint32_t n_groups, uint32_t topk_groups, uint32_t flags, float scale) {
    MX_REQUIRE_PTR(logits); MX_REQUIRE_PTR(topk_idx); MX_REQUIRE_PTR(topk_w);
    // four tokens a workgroup of 256 threads, and a launch holds fewer than 2^32
    MX_REQUIRE_SHAPE(n_tokens > 0 && n_tokens <= (1u << 26) - 4 && n_experts > 0 && n_experts <= 1024 && n_groups > 0 && n_groups <= 64 && n_experts % n_groups == 0);
    const uint32_t size = n_experts / n_groups;
    MX_REQUIRE_SHAPE(topk_groups > 0 && topk_groups <= n_groups && k > 0 && k <= (uint32_t)kMaxTopK && k <= topk_groups * size && flags < 16u);
    MX_REQUIRE_ALIGN(logits, flags & MX_ROUTE_F32 ? 4 : 2); MX_REQUIRE_ALIGN(bias, 4); MX_REQUIRE_ALIGN(topk_idx, 4); MX_REQUIRE_ALIGN(topk_w, 2);
    RouteArgs a = {logits, bias, topk_idx, reinterpret_cast<half_t*>(topk_w), n_tokens, n_experts, k, n_groups, size, size > 1 ? 0xFFFFFFFFu / size + 1u : 0u, topk_groups, 1, flags, scale, false};
    while (a.lanes * 2 * n_groups <= 64) a.lanes *= 2;
    const uint32_t per_lane = n_experts <= 64 ? 1 : n_experts <= 128 ? 2 : n_experts <= 256 ? 4 : n_experts <= 512 ? 8 : 16;
    a.wide = n_experts % per_lane == 0 && aligned(logits, per_lane * (flags & MX_ROUTE_F32 ? 4 : 2));
    const dim3 grid((n_tokens + 3) / 4), block(256);
    hipStream_t st = as_stream(s);
    if (n_experts <= 64) hipLaunchKernelGGL((route_kernel<1>), grid, block, 0, st, a);
    else if (n_experts <= 128) hipLaunchKernelGGL((route_kernel<2>), grid, block, 0, st, a);
    else if (n_experts <= 256) hipLaunchKernelGGL((route_kernel<4>), grid, block, 0, st, a);
    else if (n_experts <= 512) hipLaunchKernelGGL((route_kernel<8>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((route_kernel<16>), grid, block, 0, st, a);
    return launch_status();
}

int mx_moe_build_pack_decode(mx_stream_t s, const int32_t* topk_idx, const uint16_t* topk_w, uint32_t* expert_offsets, int32_t* sorted_idx,
                             int32_t* tk_to_packed, uint16_t* weights_packed, uint32_t E, uint32_t K) {
    MX_REQUIRE_PTR(topk_idx); MX_REQUIRE_PTR(topk_w); MX_REQUIRE_PTR(expert_offsets); MX_REQUIRE_PTR(sorted_idx); MX_REQUIRE_PTR(tk_to_packed);
    MX_REQUIRE_PTR(weights_packed);
    MX_REQUIRE_SHAPE(E > 0 && K > 0);
    hipLaunchKernelGGL(pack_decode_kernel, dim3(1), dim3(256), 0, as_stream(s), topk_idx, reinterpret_cast<const half_t*>(topk_w), expert_offsets, sorted_idx,
                       tk_to_packed, reinterpret_cast<half_t*>(weights_packed), E, K);
    return launch_status();
}

int mx_moe_build_packing_device(mx_stream_t s, const int32_t* topk_idx, const uint16_t* topk_w, uint32_t T, uint32_t K, uint32_t E, uint32_t* expert_offsets,
                                int32_t* sorted_idx, uint16_t* weights_packed, int32_t* tk_to_packed) {
    MX_REQUIRE_PTR(topk_idx); MX_REQUIRE_PTR(topk_w); MX_REQUIRE_PTR(expert_offsets); MX_REQUIRE_PTR(sorted_idx); MX_REQUIRE_PTR(tk_to_packed);
    MX_REQUIRE_PTR(weights_packed);
    MX_REQUIRE_SHAPE(E > 0 && E <= 65535 && K > 0 && T > 0 && (uint64_t)T * K <= 0x7FFFFFFFull);
    const uint32_t n = T * K, waves = n <= 256 ? 4u : n <= 2048 ? 8u : 16u, slots = (n + 64u * waves - 1u) / (64u * waves);   // a lane's
    hipStream_t st = as_stream(s);
#define MX_PACK(R, Q) \
    hipLaunchKernelGGL((pack_kernel<R, Q>), dim3((E + Q - 1u) / Q), dim3(64u * waves), 0, st, topk_idx, topk_w, n, K, E, expert_offsets, sorted_idx, weights_packed, tk_to_packed)
    if (E <= 128u) {
        if (slots <= 4u) MX_PACK(4, 1);
        else if (slots <= 16u) MX_PACK(16, 1);
        else MX_PACK(0, 1);
    } else {
        if (slots <= 4u) MX_PACK(4, 4);
        else if (slots <= 16u) MX_PACK(16, 4);
        else MX_PACK(0, 4);
    }
#undef MX_PACK
    return launch_status();
}

}  // extern "C"
